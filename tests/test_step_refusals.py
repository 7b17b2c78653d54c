"""The entry points of a token's step refuse what their kernels do not cover before any
GPU is touched: the messages, on the CPU; the rotary frequencies, which the host forms."""
import ctypes
import math

import numpy as np
import pytest

import omnivoice_amd as ov

HERE = 0x10000  # an aligned address that a refused call never reads
NAN, INF = float("nan"), float("inf")


def answer(fn, *args):
    err = ctypes.create_string_buffer(256)
    return getattr(ov.lib(), fn)(*args, err, len(err)), err.value.decode()


def refused(fn, *args):
    status, message = answer(fn, *args)
    assert status == ov.OVG_ERROR
    return message


def norm(call=refused, x=HERE, xs=64, xt=0, r=None, rs=64, t=None, ts=64, rt=2, w=HERE, o=HERE,
         os=64, ot=0, scales=None, rows=4, width=64, eps=1e-6):
    return call("ovg_op_add_rmsnorm", x, xs, xt, r, rs, t, ts, rt, w, o, os, ot, scales, rows,
                width, eps, None)


def test_norm_refuses():
    assert norm(x=None) == "add rmsnorm: null pointer"
    for name in ("w", "o"):
        assert "null" in norm(**{name: None})
    assert "rows" in norm(rows=-1)
    assert "rows" in norm(rows=2 ** 22 + 1)
    assert "width" in norm(width=0)
    assert "width" in norm(width=65537, xs=70000, os=70000)
    assert "type" in norm(xt=3)
    assert "type" in norm(xt=-1)
    assert "type" in norm(ot=4)
    assert "stride" in norm(xs=63)
    assert "stride" in norm(os=0)
    assert "go together" in norm(r=HERE)
    assert "go together" in norm(t=HERE)
    assert "stride" in norm(r=HERE, t=HERE, rs=63)
    assert "stride" in norm(r=HERE, t=HERE, ts=63)
    assert "residual" in norm(r=HERE, t=HERE, rt=1)
    assert "type" in norm(r=HERE, t=HERE, rt=3)
    assert "scales" in norm(ot=3)
    assert "scales" in norm(scales=HERE)
    for eps in (0.0, -1.0, NAN, INF):
        assert "epsilon" in norm(eps=eps)
    assert norm(answer, rows=0, x=None, w=None, o=None)[0] == ov.OVG_OK


def quantize(call=refused, x=HERE, xs=64, g=None, gs=64, kind=0, c=HERE, cs=64, s=HERE, rows=4,
             width=64):
    return call("ovg_op_quantize8", x, xs, g, gs, kind, c, cs, s, rows, width, None)


def test_quantize_refuses():
    assert quantize(x=None) == "quantize8: null pointer"
    assert "null" in quantize(c=None)
    assert "null" in quantize(s=None)
    assert "rows" in quantize(rows=-1)
    assert "rows" in quantize(rows=2 ** 22 + 1)
    assert "width" in quantize(width=0)
    assert "width" in quantize(width=65537, xs=70000, cs=70000)
    assert "type" in quantize(kind=3)
    assert "stride" in quantize(xs=63)
    assert "stride" in quantize(cs=63)
    assert "stride" in quantize(g=HERE, gs=63)
    assert quantize(answer, rows=0, x=None, c=None, s=None)[0] == ov.OVG_OK


def linear(call=refused, x=HERE, xs=64, xf=HERE, w=HERE, wf=HERE, y=HERE, ys=32, kind=1, rows=4,
           width=64, out=32):
    return call("ovg_op_linear8", x, xs, xf, w, wf, y, ys, kind, rows, width, out, None)


def test_linear_refuses():
    assert linear(x=None) == "linear8: null pointer"
    for name in ("xf", "w", "wf", "y"):
        assert "null" in linear(**{name: None})
    assert "rows" in linear(rows=-1)
    assert "rows" in linear(rows=2 ** 22 + 1)
    for width in (0, 8, 72, 65552):
        assert "multiple of 16" in linear(width=width, xs=70000)
    assert "out" in linear(out=-1)
    assert "out" in linear(out=2 ** 22 + 1, ys=2 ** 23)
    assert "type" in linear(kind=3)
    assert "stride" in linear(xs=48)
    assert "multiple of 16" in linear(xs=72)
    assert "stride" in linear(ys=31)
    assert "aligned" in linear(x=HERE + 8)
    assert "aligned" in linear(w=HERE + 1)
    assert linear(answer, rows=0, x=None)[0] == ov.OVG_OK
    assert linear(answer, out=0, w=None)[0] == ov.OVG_OK


def rotary(call=refused, q=HERE, qo=HERE, qs=1024, qos=1024, heads=8, k=HERE, ko=HERE, ks=256,
           kos=256, kv=2, kind=0, rows=4, dim=128, rot=128, f=HERE, m=1.0, pos=HERE, seq=None,
           qn=None, kn=None, eps=1e-6):
    return call("ovg_op_rotary", q, qo, qs, qos, heads, k, ko, ks, kos, kv, kind, rows, dim, rot,
                f, m, 0, pos, seq, qn, kn, eps, None)


def sequences(**over):
    f = dict(tables=None, lengths=HERE, begins=HERE, count=2, table_width=1, rows=4)
    f.update(over)
    return ov._KvSequences(**f)


def test_rotary_refuses():
    assert rotary(q=None) == "rotary: null pointer"
    for name in ("qo", "k", "ko", "f"):
        assert "null" in rotary(**{name: None})
    assert "rows" in rotary(rows=-1)
    assert "rows" in rotary(rows=2 ** 24 + 1)
    for dim in (0, 1, 127, 514):
        assert "head_dim" in rotary(dim=dim, rot=2)
    for rot in (0, 3, 130):
        assert "rotary" in rotary(rot=rot)[8:]
    assert "heads" in rotary(heads=0)
    assert "heads" in rotary(heads=4097, qs=2 ** 20, qos=2 ** 20)
    assert "heads" in rotary(kv=-1)
    assert "type" in rotary(kind=3)
    assert "magnitude" in rotary(m=INF)
    assert "magnitude" in rotary(m=NAN)
    assert "epsilon" in rotary(qn=HERE, eps=0.0)
    assert "epsilon" in rotary(kn=HERE, eps=NAN)
    for name in ("qs", "qos", "ks", "kos"):
        assert "stride" in rotary(**{name: 255})
    assert "either" in rotary(pos=None)
    assert "either" in rotary(seq=sequences())
    assert "others" in rotary(pos=None, seq=sequences(rows=5))
    assert "count" in rotary(pos=None, seq=sequences(count=-1))
    assert "count" in rotary(pos=None, seq=sequences(count=2 ** 21))
    assert "null" in rotary(pos=None, seq=sequences(begins=None))
    assert "null" in rotary(pos=None, seq=sequences(lengths=None))
    assert rotary(answer, rows=0, q=None, k=None)[0] == ov.OVG_OK
    assert rotary(answer, pos=None, seq=sequences(count=0, lengths=None, begins=None))[0] == \
        ov.OVG_OK


def sample(call=refused, z=HERE, u=None, rows=4, vocab=100, stride=100, us=100, g=0.0, mask=-1,
           setting=None, r=HERE, t=HERE, kind=2, space=None, size=0, **numbers):
    if setting is None:
        n = dict(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0)
        n.update(numbers)
        setting = ov._Sampling(**n)
    return call("ovg_op_sample", z, u, rows, vocab, stride, us, g, mask, setting or None, r, t,
                kind, space, size, None)


def test_sample_refuses():
    assert sample(z=None) == "sample: null pointer"
    assert "null" in sample(r=None)
    assert "null" in sample(t=None)
    assert "null" in sample(setting=False)
    assert "rows" in sample(rows=-1)
    assert "rows" in sample(rows=2 ** 22 + 1)
    assert "vocab" in sample(vocab=0)
    assert "vocab" in sample(vocab=2 ** 31, stride=2 ** 32)
    assert "mask_id" in sample(mask=-2)
    assert "mask_id" in sample(mask=2 ** 31)
    assert "guidance" in sample(g=INF)
    assert "stride" in sample(stride=99)
    assert "stride" in sample(u=HERE, us=99)
    assert "type" in sample(kind=3)
    for name in ("temperature", "top_p", "min_p"):
        assert name in sample(**{name: NAN})
    assert sample(answer, rows=0, z=None, r=None, t=None)[0] == ov.OVG_OK
    need = ov.op_sample_workspace(4, 9000)
    assert need > 0 and ov.op_sample_workspace(4, 2048) == 0
    for args in ((-1, 100), (2 ** 22 + 1, 100), (4, 0), (4, 2 ** 31)):
        assert ov.op_sample_workspace(*args) == -1


@pytest.mark.parametrize("stream", [None, 0, HERE])
def test_host_tensors_are_refused(stream):
    torch = pytest.importorskip("torch")
    x, w = torch.zeros(4, 64), torch.zeros(64)
    codes, scales = torch.zeros(4, 64, dtype=torch.uint8), torch.zeros(4)
    q, f = torch.zeros(4, 2, 64), torch.zeros(32)
    ints = torch.zeros(4, dtype=torch.int32)
    for call in (lambda: ov.op_add_rmsnorm(x, w, x, stream=stream),
                 lambda: ov.op_quantize8(x, codes, scales, stream=stream),
                 lambda: ov.op_linear8(codes, scales, codes, scales, torch.zeros(4, 4),
                                       stream=stream),
                 lambda: ov.op_rotary(q, q, None, None, f, positions=ints, stream=stream),
                 lambda: ov.op_sample(x, scales, ints, stream=stream)):
        with pytest.raises(ov.GeneratorError, match="needs tensors of a GPU, got cpu"):
            call()


def test_python_checks_of_tensors():
    torch = pytest.importorskip("torch")
    x, w = torch.zeros(4, 64), torch.zeros(64)
    codes, scales = torch.zeros(4, 64, dtype=torch.uint8), torch.zeros(4)
    q, f = torch.zeros(4, 2, 64), torch.zeros(32)
    ints = torch.zeros(4, dtype=torch.int32)
    bad = [
        (lambda: ov.op_add_rmsnorm(x, w[:63], x), "weight"),
        (lambda: ov.op_add_rmsnorm(x, w, x[:3]), "out"),
        (lambda: ov.op_add_rmsnorm(x.t(), w[:4], x.t()), "x: needs"),
        (lambda: ov.op_add_rmsnorm(x, w, x, total=x), "residual"),
        (lambda: ov.op_add_rmsnorm(x, w, x, residual=x, total=x.half()), "differ"),
        (lambda: ov.op_add_rmsnorm(x, w, x, scales=scales), "8 bits"),
        (lambda: ov.op_add_rmsnorm(x, w, codes), "without scales"),
        (lambda: ov.op_add_rmsnorm(x, w, codes, scales=scales[:3]), "scales"),
        (lambda: ov.op_quantize8(x, x, scales), "codes"),
        (lambda: ov.op_quantize8(x, codes, scales, gate=x.half()), "differ"),
        (lambda: ov.op_quantize8(x, codes, scales, gate=x[:, :60]), "gate"),
        (lambda: ov.op_quantize8(ints[:, None], codes, scales), "not supported"),
        (lambda: ov.op_linear8(x, scales, codes, scales, x), "not supported"),
        (lambda: ov.op_linear8(codes, scales, codes[:, :32], scales, torch.zeros(4, 4)), "w: "),
        (lambda: ov.op_linear8(codes, scales, codes, scales, torch.zeros(4, 5)), "y: "),
        (lambda: ov.op_linear8(codes, scales[:2], codes, scales, torch.zeros(4, 4)), "x_scales"),
        (lambda: ov.op_rotary(q, q, q, None, f, positions=ints), "go together"),
        (lambda: ov.op_rotary(q, q.half(), None, None, f, positions=ints), "differ"),
        (lambda: ov.op_rotary(q, q, None, None, f), "either"),
        (lambda: ov.op_rotary(q, q, None, None, f, positions=ints[:2]), "positions"),
        (lambda: ov.op_rotary(q, q, None, None, f.double(), positions=ints), "frequencies"),
        (lambda: ov.op_rotary(q, q, None, None, f, positions=ints, q_norm=f), "q_norm"),
        (lambda: ov.op_rotary(q.transpose(0, 1), q, None, None, f, positions=ints), "q: needs"),
        (lambda: ov.op_sample(x, scales, ints.long()), "tokens"),
        (lambda: ov.op_sample(x, scales[:3], ints), "random"),
        (lambda: ov.op_sample(x, scales, ints, top_k=scales), "top_k"),
        (lambda: ov.op_sample(x, scales, ints, temperature=scales[:2]), "temperature"),
        (lambda: ov.op_sample(x, scales, ints, top_k=2 ** 31), "top_k"),
        (lambda: ov.op_sample(x, scales, ints, uncond=x.half()), "uncond"),
        (lambda: ov.op_sample(x[0], scales, ints), "logits")]
    for call, word in bad:
        with pytest.raises(ov.GeneratorError, match=word):
            call()


# ------------------------------------------------------------------ frequencies

def test_frequencies():
    f, m = ov.rotary_frequencies(128, 1e6)
    i = np.arange(64)
    np.testing.assert_array_equal(f, (1e6 ** (-i / 64)).astype(np.float32))
    assert m == 1.0
    g, m = ov.rotary_frequencies(128, 1e6, "linear", 4.0)
    np.testing.assert_array_equal(g, (1e6 ** (-i / 64) / 4).astype(np.float32))
    assert m == 1.0
    g, m = ov.rotary_frequencies(128, 1e6, "base", 4.0)
    assert g[0] == 1.0 and m == 1.0
    assert abs(g[-1] * 4 / f[-1] - 1) < 1e-6
    assert ov.rotary_frequencies(2, 1e6, "base", 4.0)[0].tolist() == [1.0]


def test_frequencies_by_parts():
    f, _ = ov.rotary_frequencies(128, 1e6)
    g, m = ov.rotary_frequencies(128, 1e6, "parts", 8.0, 32768)
    assert m == np.float32(0.1 * math.log(8.0) + 1)
    turns = 32768 * f.astype(np.float64) / (2 * math.pi)
    ratio = g.astype(np.float64) / f
    # Whole pairs around the two borders belong to the ramp.
    step = 1e6 ** (1 / 64)
    assert (np.abs(ratio[turns > 32 * step] - 1) < 1e-6).all()
    assert (np.abs(ratio[turns < 1 / step] * 8 - 1) < 1e-6).all()
    assert (np.diff(ratio) <= 1e-7).all()
    assert ((ratio > 0.2) & (ratio < 0.9)).any()
    same, m = ov.rotary_frequencies(128, 1e6, "parts", 1.0, 32768)
    np.testing.assert_array_equal(same, f)
    assert m == 1.0


@pytest.mark.parametrize("original", [1.0, 3.0, 6.0])
def test_frequencies_by_parts_of_less_than_a_turn(original):
    """Trained on fewer positions than the first pair turns in once (2 pi): every pair is
    divided, the first one too."""
    for rotary, theta in ((128, 1e6), (2, 1e4), (64, 2.0)):
        f, _ = ov.rotary_frequencies(rotary, theta)
        g, _ = ov.rotary_frequencies(rotary, theta, "parts", 8.0, original)
        np.testing.assert_array_equal(g, f / 8)


def test_frequencies_refuse():
    for args in ((0,), (3,), (-2,), (514,), (128, 1.0), (128, NAN), (128, INF),
                 (128, 1e6, "linear", 0.5), (128, 1e6, "base", NAN), (128, 1e6, "base", INF),
                 (128, 1e6, "parts", 2.0), (128, 1e6, "parts", 2.0, NAN),
                 (128, 1e6, "yarn", 2.0)):
        with pytest.raises(ov.GeneratorError):
            ov.rotary_frequencies(*args)


def test_the_most_rows():
    """What a launch cannot count is refused before any device work."""
    assert "rows" in norm(rows=2 ** 22)
    assert "rows" in quantize(rows=2 ** 22)
    assert "rows" in linear(rows=2 ** 22)
    assert "out" in linear(out=2 ** 22, ys=2 ** 22)
    assert "rows" in rotary(rows=2 ** 24)
    assert "rows" in sample(rows=2 ** 22)
    assert "rows times vocab" in sample(rows=2 ** 21, vocab=40000, stride=40000)
    assert ov.op_sample_workspace(2 ** 21, 40000) == -1
    assert ov.op_sample_workspace(2 ** 21, 2048) == 0
    assert ov.op_sample_workspace(2 ** 20, 40000) > 0
    assert ov.op_sample_workspace(63, 2 ** 30) > 0
    assert ov.op_sample_workspace(64, 2 ** 30) == -1


def test_a_workspace_that_does_not_fit():
    need = ov.op_sample_workspace(4, 9000)
    for space, size in ((None, need), (HERE, need - 1), (HERE, 0)):
        assert f"workspace of {need} bytes" in sample(vocab=9000, stride=9000, space=space,
                                                      size=size)
    assert "16-byte aligned" in sample(vocab=9000, stride=9000, space=HERE + 8, size=need)
