"""Refusals of tqk_decode_q8_weights, tqk_evict_q8 and tqk_process_logits, which all come before any device work, the
argument structs' layouts, and the plain implementations' own checks -- without a GPU."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

from _cache_ops import attend64, evict_ref, logits_ref, pack_bits, weight_bound

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
FAKE = 4096  # an aligned address that nothing touches


@pytest.fixture(scope="module")
def tqk():
    from tailorquantkernel_b200 import tqk as t
    return t


@pytest.mark.parametrize("struct,c_name", [("WeightsArgs", "tqk_weights_args"), ("EvictArgs", "tqk_evict_args"),
                                           ("LogitsArgs", "tqk_logits_args")])
def test_struct_layouts_match_c(tqk, tmp_path, struct, c_name):
    cls = getattr(tqk, struct)
    fields = [f for f, _ in cls._fields_]
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "tqk.h"\nint main(void){\n'
                   f'printf("%zu\\n", sizeof({c_name}));\n' +
                   "".join(f'printf("%zu\\n", offsetof({c_name}, {f}));\n' for f in fields) + "return 0;}\n")
    exe = tmp_path / "layout"
    subprocess.run(["/usr/bin/gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    vals = [int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert vals == [ctypes.sizeof(cls)] + [getattr(cls, f).offset for f in fields]


def _fill(struct, good, change):
    for k, v in {**good, **change}.items():
        setattr(struct, k, v)
    return struct


DECODE = dict(k=FAKE, v=FAKE, q=FAKE, out=FAKE, n_items=2, n_q_heads=8, n_kv_heads=2, head_dim=128, max_tokens=64,
              item_stride=2 * 64 * 4, len0=10)
WEIGHTS = dict(weight=FAKE, weight_out=FAKE, item_stride=2 * 64)


@pytest.mark.parametrize("decode,weights,status", [
    ({}, dict(weight=None), "EINVAL"), ({}, dict(weight_out=None), "EINVAL"),
    ({}, dict(weight=FAKE + 2), "EALIGN"), ({}, dict(weight_out=FAKE + 1), "EALIGN"),
    (dict(out_mode=1), {}, "EINVAL"),                      # partial output has no weights yet
    ({}, dict(item_stride=127), "EINVAL"), ({}, dict(item_stride=0), "EINVAL"),
    ({}, dict(position=FAKE), "EINVAL"),                   # positions belong to appended rows
    (dict(k_new=FAKE, v_new=FAKE), dict(new_pos=FAKE), "EINVAL"),
    (dict(k_new=FAKE), {}, "EINVAL"), (dict(n_q_heads=7), {}, "EINVAL"), (dict(head_dim=96), {}, "EUNSUPPORTED"),
    (dict(k=FAKE + 8), {}, "EALIGN"), (dict(len0=65), {}, "EPOS"), (dict(len0=0, k_new=FAKE, v_new=FAKE), {}, "EPOS"),
    (dict(lens=FAKE, max_len=65), {}, "EINVAL"), (dict(q_norm=FAKE), {}, "EINVAL"), (dict(rope_cos=FAKE), {}, "EINVAL"),
    (dict(n_items=0), {}, "EINVAL"), (dict(q=None), {}, "EINVAL"),
])
def test_decode_weights_refusals(tqk, decode, weights, status):
    a, w = _fill(tqk.DecodeArgs(), DECODE, decode), _fill(tqk.WeightsArgs(), WEIGHTS, weights)
    assert tqk.tqk_decode_q8_weights(ctypes.byref(a), ctypes.byref(w), None, 0, None) == getattr(tqk, status)
    assert tqk.tqk_last_error()


def test_null_structs(tqk):
    a, w = tqk.DecodeArgs(), tqk.WeightsArgs()
    assert tqk.tqk_decode_q8_weights(None, ctypes.byref(w), None, 0, None) == tqk.EINVAL
    assert tqk.tqk_decode_q8_weights(ctypes.byref(a), None, None, 0, None) == tqk.EINVAL
    assert tqk.tqk_decode_weights_workspace_size(None, None) == tqk.EINVAL
    assert tqk.tqk_evict_q8(None, None) == tqk.EINVAL
    assert tqk.tqk_process_logits(None, None) == tqk.EINVAL


EVICT = dict(k=FAKE, v=FAKE, weight=FAKE, weight_out=FAKE, position=FAKE, position_out=FAKE, n_items=2, n_kv_heads=2,
             head_dim=128, max_tokens=64, item_stride=2 * 64 * 4, stat_item_stride=2 * 64, len0=60, budget=32, n_first=4,
             n_recent=8)


@pytest.mark.parametrize("change,status", [
    (dict(k=None), "EINVAL"), (dict(weight_out=None), "EINVAL"), (dict(position_out=None), "EINVAL"),
    (dict(position=None, position_out=None), "EINVAL"),    # protected positions need positions
    (dict(n_items=0), "EINVAL"), (dict(head_dim=48), "EINVAL"), (dict(head_dim=160), "EUNSUPPORTED"),
    (dict(budget=0), "EINVAL"), (dict(budget=65), "EINVAL"), (dict(n_first=25), "EINVAL"), (dict(n_first=-1), "EINVAL"),
    (dict(n_recent=2 ** 31 - 1), "EINVAL"), (dict(item_stride=511), "EINVAL"), (dict(stat_item_stride=127), "EINVAL"),
    (dict(len0=65), "EPOS"), (dict(len0=-1), "EPOS"), (dict(len_step=5), "EPOS"), (dict(lens=FAKE, max_len=65), "EINVAL"),
    (dict(lens=FAKE, max_len=-1), "EINVAL"), (dict(k=FAKE + 4), "EALIGN"), (dict(item_stride=513), "EALIGN"),
    (dict(head_dim=64, k=FAKE + 2), "EALIGN"), (dict(weight=FAKE + 2), "EALIGN"), (dict(position_out=FAKE + 1), "EALIGN"),
    (dict(n_items=1, max_tokens=600000, len0=258049), "EUNSUPPORTED"),
    (dict(n_items=70000), "EINVAL"),
])
def test_evict_refusals(tqk, change, status):
    assert tqk.tqk_evict_q8(ctypes.byref(_fill(tqk.EvictArgs(), EVICT, change)), None) == getattr(tqk, status)
    assert tqk.tqk_last_error()


LOGITS = dict(logits=FAKE, out=FAKE * 2, choice=FAKE, n_rows=2, vocab_size=100, tokens=FAKE, token_offsets=FAKE, n_tokens=5,
              repetition=FAKE, bias_tokens=FAKE, bias_values=FAKE, bias_offsets=FAKE, n_bias=3, mask=FAKE, n_mask_rows=2)


@pytest.mark.parametrize("change,status", [
    (dict(logits=None), "EINVAL"), (dict(out=None, choice=None), "EINVAL"), (dict(n_rows=0), "EINVAL"),
    (dict(vocab_size=0), "EINVAL"), (dict(n_rows=70000, n_mask_rows=70000), "EINVAL"),
    (dict(vocab_size=2 ** 29), "EUNSUPPORTED"), (dict(n_tokens=2 ** 29), "EUNSUPPORTED"),
    (dict(logits_stride=99), "EINVAL"), (dict(out_stride=99), "EINVAL"), (dict(out=FAKE, out_stride=101), "EINVAL"),
    (dict(tokens=None), "EINVAL"), (dict(token_offsets=None), "EINVAL"), (dict(n_tokens=-1), "EINVAL"),
    (dict(bias_values=None), "EINVAL"), (dict(bias_offsets=None), "EINVAL"), (dict(bias_tokens=None), "EINVAL"),
    (dict(n_bias=-1), "EINVAL"), (dict(mask_stride=3), "EINVAL"), (dict(n_mask_rows=1), "EINVAL"),
    (dict(mask=None, mask_rows=FAKE), "EINVAL"), (dict(logits=FAKE + 2), "EALIGN"), (dict(mask=FAKE + 1), "EALIGN"),
])
def test_logits_refusals(tqk, change, status):
    assert tqk.tqk_process_logits(ctypes.byref(_fill(tqk.LogitsArgs(), LOGITS, change)), None) == getattr(tqk, status)
    assert tqk.tqk_last_error()


def test_python_helpers_refuse_wrong_types(tqk):
    """Index arrays of another type than int32, or sums of another than fp32, would be misread: refused by name."""
    import torch
    f, i = torch.zeros(4), torch.zeros(4, dtype=torch.int64)
    with pytest.raises(ValueError, match="CUDA"):
        tqk.weights_args(f)
    with pytest.raises(ValueError, match="CUDA"):
        tqk.logits_args(torch.zeros(2, 3))
    with pytest.raises(ValueError, match="int32"):
        tqk.weights_args(FAKE, position=i)
    with pytest.raises(ValueError, match="float32"):
        tqk.weights_args(f.double())
    with pytest.raises(ValueError, match="int32"):
        tqk.evict_args(FAKE, FAKE, 1, 32, 4, 2, weight=FAKE, lens=i)
    with pytest.raises(ValueError, match="float32"):
        tqk.logits_args(torch.zeros(2, 3, dtype=torch.bfloat16))


class _FakeTensor:
    """What the helpers look at of a CUDA tensor, without a GPU."""

    def __init__(self, device, dtype="float32"):
        self.device, self.dtype, self.is_cuda = type("D", (), {"index": device}), f"torch.{dtype}", True

    def is_contiguous(self):
        return True

    def data_ptr(self):
        return FAKE


def test_python_helpers_refuse_tensors_of_another_device(tqk, monkeypatch):
    """The library launches on the current device; a call's tensors must share it."""
    import torch
    with pytest.raises(ValueError, match="several devices"):
        tqk.weights_args(_FakeTensor(0), _FakeTensor(1))
    w = tqk.weights_args(_FakeTensor(1))
    e = tqk.evict_args(_FakeTensor(1), _FakeTensor(1), 1, 32, 4, 2, weight=_FakeTensor(1))
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    with pytest.raises(ValueError, match="cuda:1"):
        tqk.decode_weights(tqk.DecodeArgs(), w)
    with pytest.raises(ValueError, match="cuda:1"):
        tqk.evict(e)


def test_plain_eviction():
    """The plain implementation on a case worked out by hand."""
    w = np.array([5, 1, 4, np.nan, 3, 3, 0.5, 9], np.float32)
    p = np.arange(8, dtype=np.int32)
    keep, dst, src = evict_ref(w, p, 8, 4, 1, 2)       # protected: 0, 6, 7; then the largest of the rest: 2
    assert np.flatnonzero(keep).tolist() == [0, 2, 6, 7] and dst.tolist() == [1, 3] and src.tolist() == [6, 7]
    keep, dst, src = evict_ref(w, None, 8, 5, 0, 0)    # 9, 5, 4, then the lower of the two threes
    assert np.flatnonzero(keep).tolist() == [0, 2, 4, 5, 7] and dst.tolist() == [1, 3] and src.tolist() == [5, 7]
    keep, dst, src = evict_ref(w, None, 8, 4, 0, 0)
    assert np.flatnonzero(keep).tolist() == [0, 2, 4, 7] and dst.tolist() == [1, 3] and src.tolist() == [4, 7]


def test_plain_logits():
    x = np.array([2, -2, 0, 1, 5], np.float32)
    y, best = logits_ref(x, tokens=np.array([0, 1, 1, 9, -1], np.int32), prompt=1, repetition=2.0, frequency=0.5,
                         presence=0.25, bias=[(3, 1.0), (3, 2.0), (7, 100.0)], allowed=np.array([1, 1, 1, 1, 0], bool))
    assert y.tolist() == [1.0, -4.0 - 1.0 - 0.25, 0.0, 4.0, -np.inf] and best == 3
    assert logits_ref(x, allowed=np.zeros(5, bool))[1] == -1
    assert pack_bits(np.array([[0] * 31 + [1, 1]], bool)).view(np.uint32).tolist() == [[2 ** 31, 1]]


def test_plain_attention_sums_to_one_per_head():
    import oracle
    rng = np.random.default_rng(0)
    port = oracle.Oracle("port")
    q, k, v = (port.quantize_rows(rng.standard_normal(s, dtype=np.float32)) for s in ((2, 6, 64), (2, 2, 9, 64), (2, 2, 9, 64)))
    _, w, big = attend64(q, k, v, [9, 4])
    assert np.allclose(w.sum(-1), 3.0) and (w[1, :, 4:] == 0).all() and 0 < weight_bound(2, big, 9) < 1e-5


def test_library_buffers_of_the_per_thread_stream_belong_to_a_thread(tmp_path):
    """The key of the library-owned workspaces: one handle, cudaStreamPerThread, is another stream in every thread."""
    from tailorquantkernel_b200 import build
    src, exe = tmp_path / "key.cpp", tmp_path / "key"
    src.write_text('#include <cstdio>\n#include <set>\n#include <thread>\n#include <vector>\n#include "tqk_stream_key.h"\n'
                   "using namespace tqk;\n"
                   "int main() {\n"
                   "  cudaStream_t own = reinterpret_cast<cudaStream_t>(64);\n"
                   "  std::vector<StreamKey> got(16, StreamKey{});\n"
                   "  // one thread after the other, so that their ids may be the same\n"
                   "  for (int i = 0; i < 8; i++) std::thread([&, i] {\n"
                   "    got[2 * i] = stream_key(i % 2, cudaStreamPerThread);\n"
                   "    got[2 * i + 1] = stream_key(i % 2, own);\n"
                   "    StreamKey again = stream_key(i % 2, cudaStreamPerThread);\n"
                   "    if (again < got[2 * i] || got[2 * i] < again) got[2 * i + 1].thread = 99;\n"
                   "  }).join();\n"
                   "  std::set<StreamKey> keys(got.begin(), got.end());\n"
                   '  std::printf("%zu", keys.size());\n'
                   "}\n")
    cuda = os.path.dirname(os.path.dirname(build._nvcc()))
    subprocess.run(["/usr/bin/g++", "-std=c++17", "-pthread", "-I", build.CSRC, "-I", os.path.join(cuda, "include"), str(src),
                    "-o", str(exe)], check=True)
    # 8 threads' own streams, and one other stream on each of two devices
    assert subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout == "10"


def test_logit_clusters_fit_the_device(tmp_path):
    """CTAs per row: never more than the device holds in a cluster, and otherwise the measured choices."""
    from tailorquantkernel_b200 import build
    src, exe = tmp_path / "plan.cpp", tmp_path / "plan"
    src.write_text('#include <cstdio>\n#include <cstdlib>\n#include "tqk_logits_plan.h"\n'
                   "int main(int n, char **v) {\n"
                   "  for (int i = 1; i + 3 < n; i += 4)\n"
                   '    std::printf("%d ", 1 << tqk::logits_cluster_log(atoi(v[i]), atoi(v[i + 1]), atoi(v[i + 2]), atoi(v[i + 3])));\n'
                   "}\n")
    subprocess.run(["/usr/bin/g++", "-std=c++17", "-I", build.CSRC, str(src), "-o", str(exe)], check=True)

    def ctas(*cases):
        got = subprocess.run([str(exe)] + [str(x) for c in cases for x in c], capture_output=True, text=True, check=True)
        return [int(x) for x in got.stdout.split()]

    rows = [1, 2, 7, 18, 19, 37, 74, 148, 256, 512, 65535]
    vocabs = [1, 4096, 4097, 8192, 8193, 16385, 32003, 65537, 128256, 262144, 2 ** 29 - 1]
    for sms in (148, 16, 1):
        cases = [(r, v, sms) for r in rows for v in vocabs]
        wide, narrow = ctas(*((*c, 16) for c in cases)), ctas(*((*c, 8) for c in cases))
        assert max(narrow) <= 8 and all(n == min(w, 8) for w, n in zip(wide, narrow))
    assert ctas((1, 128256, 148, 16), (37, 128256, 148, 16), (256, 128256, 148, 16), (512, 30001, 148, 16),
                (512, 8001, 148, 16), (10, 30001, 148, 16), (7, 4096, 148, 16)) == [16, 8, 8, 2, 1, 8, 1]


def test_decode_args_keep_and_check_their_tensors(tqk, monkeypatch):
    """The struct holds bare addresses, so it keeps its tensors alive; a decode with weights refuses tensors of another
    device wherever they are, and lengths that are not int32."""
    import gc
    import weakref

    import torch
    a = tqk.decode_args(_FakeTensor(1), _FakeTensor(1), 8, 2, 128, 64, _FakeTensor(1), _FakeTensor(1),
                        lens=_FakeTensor(1, "int32"), k_new=_FakeTensor(1), v_new=_FakeTensor(1), q_norm=_FakeTensor(1),
                        k_norm=_FakeTensor(1), rope_cos=_FakeTensor(1), rope_sin=_FakeTensor(1))
    seen = [weakref.ref(t) for t in a._keep]
    gc.collect()
    assert len(seen) == 11 and all(r() is not None for r in seen)
    del a
    gc.collect()
    assert all(r() is None for r in seen)
    with pytest.raises(ValueError, match="int32"):
        tqk.decode_args(FAKE, FAKE, 8, 2, 128, 64, FAKE, FAKE, lens=_FakeTensor(0, "int64"))
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)

    def call(decode_device, weights_device):
        tqk.decode_weights(tqk.decode_args(FAKE, FAKE, 8, 2, 128, 64, FAKE, _FakeTensor(decode_device)),
                           tqk.weights_args(_FakeTensor(weights_device)))

    with pytest.raises(ValueError, match="several devices"):
        call(1, 0)
    with pytest.raises(ValueError, match="several devices"):
        call(0, 1)
    with pytest.raises(ValueError, match="cuda:1"):
        call(1, 1)
    with pytest.raises(ValueError, match="cuda:1"):
        tqk.decode_weights(tqk.decode_args(FAKE, FAKE, 8, 2, 128, 64, FAKE, _FakeTensor(1)), tqk.weights_args(FAKE))


class _FakeMatrix(_FakeTensor):
    """A fake CUDA tensor with a shape, contiguous."""

    def __init__(self, *shape, dtype="float32"):
        super().__init__(0, dtype)
        self.shape = shape

    def dim(self):
        return len(self.shape)

    def numel(self):
        return int(np.prod(self.shape))

    def stride(self, i):
        return int(np.prod(self.shape[i + 1:]))


def test_logits_args_refuse_arrays_that_are_too_short(tqk):
    """Everything the kernel indexes by row or list entry is as long as the call says."""
    i32 = dict(dtype="int32")
    good = dict(out=_FakeMatrix(3, 64), choice=_FakeMatrix(3, **i32), tokens=_FakeMatrix(9, **i32),
                token_offsets=_FakeMatrix(4, **i32), prompt_lens=_FakeMatrix(3, **i32), repetition=_FakeMatrix(3),
                frequency=_FakeMatrix(3), presence=_FakeMatrix(3), bias_tokens=_FakeMatrix(5, **i32),
                bias_values=_FakeMatrix(5), bias_offsets=_FakeMatrix(4, **i32), mask=_FakeMatrix(2, 2, **i32),
                mask_rows=_FakeMatrix(3, **i32))
    a = tqk.logits_args(_FakeMatrix(3, 64), **good)
    assert (a.n_rows, a.vocab_size, a.n_tokens, a.n_bias, a.n_mask_rows) == (3, 64, 9, 5, 2)
    for name in ("choice", "token_offsets", "prompt_lens", "repetition", "frequency", "presence", "bias_values", "bias_offsets",
                 "mask_rows"):
        short = _FakeMatrix(good[name].shape[0] - 1, dtype=str(good[name].dtype).split(".")[1])
        with pytest.raises(ValueError, match=name):
            tqk.logits_args(_FakeMatrix(3, 64), **{**good, name: short})
    for name in ("n_tokens", "n_bias"):
        with pytest.raises(ValueError, match="tokens"):
            tqk.logits_args(_FakeMatrix(3, 64), **good, **{name: 10})
    tqk.logits_args(_FakeMatrix(3, 64), tokens=_FakeMatrix(9, **i32), token_offsets=FAKE, repetition=FAKE)  # addresses
