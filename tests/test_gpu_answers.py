"""GPU tests of the answering end through graphs: fully connected layers with 8-bit weights (Graph.fp8_fc) and score().

Tolerance of a layer: the reference uses the codes and scales that the definition fixes, so only the roundings of the 32-bit sums
differ, at most 128 + blocks + 8 of one step 2^-23 of the magnitudes summed (see test_gpu_fp8_fc.py).  A layer behind another one
is checked on the values that the one in front gave, because a last-bit difference there may move a code."""
import math

import numpy as np
import pytest

import deepracin_b200 as dr
from gpu_helpers import conv_build, rel_err, run_graph

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def e4m3(v):
    e = (torch.frexp(v)[1] - 1).clamp_min(-6)
    step = torch.ldexp(torch.ones_like(v), e - 3)
    return (torch.round(v / step) * step).clamp(-448, 448)


def blocks_of(x, dims):
    """x padded with zeros to whole blocks of 128 in its last `dims` dimensions"""
    pad = []
    for d in range(dims):
        pad += [0, -x.shape[-1 - d] % 128]
    return torch.nn.functional.pad(x, pad)


def rounded(x, whole):
    """float64 values that x [rows, n] stands for: scales per row and 128 values, or per 128 x 128 (whole)"""
    r, n = x.shape
    p = blocks_of(x, 2 if whole else 1)
    p = p.view(p.shape[0] // 128, 128, -1, 128) if whole else p.view(r, -1, 128)
    a = p.abs().amax((1, 3) if whole else 2, keepdim=True).clamp_min(2.0 ** -96)
    top = torch.full((), 448.0)
    q = e4m3((p * (top / a)).double()) * (a / top).double()
    return q.view(-1, q.shape[-2] * 128 if not whole else p.shape[2] * 128)[:r, :n]


def check_layer(got, x, w, b, act):
    """x [n, nin] float32 as the layer saw it, w [nin, nout] float32"""
    xq, wq = rounded(torch.from_numpy(np.ascontiguousarray(x)), False), rounded(torch.from_numpy(np.ascontiguousarray(w)), True)
    ref, mag = xq @ wq + torch.from_numpy(b).double(), xq.abs() @ wq.abs() + torch.from_numpy(b).double().abs()
    if act:
        ref = ref.clamp_min(0)
    bound = mag * (128 + -(-x.shape[1] // 128) + 8) * 2.0 ** -23 + 1e-37
    err = (torch.from_numpy(np.ascontiguousarray(got)).double() - ref).abs()
    assert bool((err <= bound).all()), float((err / bound).max())


def weights(nin, nout, seed):
    r = np.random.RandomState(seed)
    return (r.randn(nin, nout) * (2.0 / nin) ** 0.5).astype(np.float32), r.randn(nout).astype(np.float32) * 0.1


@pytest.mark.parametrize("n,opts", [(1, {}), (3, dict(math="tf32")), (20, dict(cuda_graph=True)), (100, {}), (260, dict(math="fp32x3"))])
def test_two_layers_and_their_scores(n, opts):
    """a hidden layer and the class scores behind it, then log probabilities, entropy and top five"""
    nin, hidden, classes = 1152, 520, 1000
    w1, b1 = weights(nin, hidden, 1)
    w2, b2 = weights(hidden, classes, 2)
    labels = np.random.RandomState(n).randint(0, classes, n)
    with dr.Environment() as env:
        g = env.create_graph("CHW")
        g.batch, g.fp8_fc = n, True
        for k, v in opts.items():
            setattr(g, k, v)
        x = dr.feed_node(g, [nin, 1, 1])
        h = dr.Fully_Connected(x, [nin, hidden], "relu", w1, b1)
        y = dr.Fully_Connected(h, [hidden, classes], "linear", w2, b2)
        dr.mark_as_output(h)
        dr.mark_as_output(y)
        dr.prepare(g)
        for seed in range(2):       # the second time on other inputs, by replay where there is one
            f = np.random.RandomState(seed).randn(n, nin, 1, 1).astype(np.float32)
            dr.feed_data(x, f)
            got_h, got_y = [np.asarray(a).reshape(n, -1) for a in dr.apply(g)]
            check_layer(got_h, f.reshape(n, nin), w1, b1, 1)
            check_layer(got_y, got_h, w2, b2, 0)
            lp, ent, top, idx = dr.score(y, labels, 5)
            v = got_y.astype(np.float64)
            logp = v - np.log(np.exp(v - v.max(1, keepdims=True)).sum(1, keepdims=True)) - v.max(1, keepdims=True)
            order = np.argsort(-got_y, axis=1, kind="stable")[:, :5]
            assert np.array_equal(idx, order)
            tol = 72 * 2.0 ** -24 + 2.0 ** -21 * np.abs(logp).max()      # sums of 1000 terms, exponents of up to max |log p|
            assert np.abs(lp - logp[np.arange(n), labels]).max() <= tol
            assert np.abs(top - np.take_along_axis(logp, order, 1)).max() <= tol
            assert np.abs(ent + (np.exp(logp) * logp).sum(1)).max() <= 4 * tol
        lp2, _, top2, _ = dr.score(y, np.stack([labels, np.full(n, -1)], 1), 0, scale=0.5)
        assert lp2.shape == (n, 2) and (lp2[:, 1] == 0).all() and top2.shape == (n, 0)
        from deepracin_b200 import lib
        assert lib.dR_getDeviceStatus(g.ptr) == 0


def test_behind_a_convolution_and_against_the_float_layer():
    """the layer flattens (y, x, channel) as the float layer does; its outputs are the float layer's within the rounding of operands"""
    n, c, hw, classes = 4, 16, 8, 70
    r = np.random.RandomState(0)
    x = r.randn(n, 3, hw, hw).astype(np.float32)
    wt = (r.randn(3, c, 3, 3) * 0.2).astype(np.float32)
    b = r.randn(c).astype(np.float32) * 0.1
    w, bf = weights(c * hw * hw, classes, 3)

    def build(g, f):
        conv = conv_build(wt, b)(g, f)
        return [conv, dr.Fully_Connected(conv, [c * hw * hw, classes], "linear", w, bf)]

    conv, out = run_graph(build, [x], fp8_fc=True)
    conv0, out0 = run_graph(build, [x])
    assert np.array_equal(conv, conv0)
    check_layer(out.reshape(n, classes), conv.transpose(0, 2, 3, 1).reshape(n, -1), w, bf, 0)
    # 4 significant bits: each operand off by up to 2^-4 of itself, so an output by 2^-3 of the magnitudes summed
    mag = np.abs(conv.transpose(0, 2, 3, 1).reshape(n, -1)).astype(np.float64) @ np.abs(w).astype(np.float64)
    assert (np.abs(out.reshape(n, classes) - out0.reshape(n, classes)) <= mag * (2 * 2.0 ** -4 + 2.0 ** -8)).all()


def test_off_by_default_and_saved_graphs_keep_float_weights(tmp_path):
    nin, nout = 256, 40
    w, b = weights(nin, nout, 4)
    f = np.random.RandomState(5).randn(2, nin, 1, 1).astype(np.float32)

    def build(g, feeds):
        return dr.Fully_Connected(feeds[0], [nin, nout], "linear", w, b)

    (plain,) = run_graph(build, [f])
    assert rel_err(plain.reshape(2, nout), f.reshape(2, nin).astype(np.float64) @ w + b) <= 1e-5
    with dr.Environment() as env:
        g = env.create_graph("CHW")
        g.batch, g.fp8_fc = 2, True
        x = dr.feed_node(g, [nin, 1, 1])
        y = build(g, [x])
        dr.mark_as_output(y)
        dr.prepare(g)
        dr.save_graph(g, str(tmp_path))
    with dr.Environment() as env:
        g = env.create_graph("CHW")
        g.batch = 2
        nodes, feeds = dr.load_graph(g, str(tmp_path / "dr_graph_export") + "/")
        dr.mark_as_output(nodes[-1])
        dr.prepare(g)
        dr.feed_data(feeds[0], f)
        (again,) = dr.apply(g)
    assert np.array_equal(np.asarray(again).reshape(2, nout), plain.reshape(2, nout))


def test_a_feed_buffer_of_the_callers_is_followed():
    """the caller replaces the device buffer that the layer reads between two applies"""
    import ctypes
    nin, nout = 640, 130
    w, b = weights(nin, nout, 6)
    r = np.random.RandomState(7)
    with dr.Environment() as env:
        g = env.create_graph("CHW")
        g.fp8_fc = True
        x = dr.feed_node(g, [nin, 1, 1])
        y = dr.Fully_Connected(x, [nin, nout], "relu", w, b)
        dr.mark_as_output(y)
        dr.prepare(g)
        for _ in range(3):
            f = r.randn(1, nin).astype(np.float32)
            t = torch.from_numpy(f).cuda()
            torch.cuda.synchronize()
            mem = ctypes.c_void_p(t.data_ptr())
            assert dr.lib.dR_setDataFeedNodeBuffer(g.ptr, x.ptr, ctypes.byref(mem))
            (out,) = dr.apply(g)
            check_layer(np.asarray(out).reshape(1, nout), f, w, b, 1)


def test_score_refuses():
    nin, nout = 64, 20
    w, b = weights(nin, nout, 8)
    with dr.Environment() as env:
        g = env.create_graph("CHW")
        g.batch = 2
        x = dr.feed_node(g, [nin, 1, 1])
        h = dr.Fully_Connected(x, [nin, nin], "relu", *weights(nin, nin, 9))
        y = dr.Fully_Connected(h, [nin, nout], "linear", w, b)
        dr.mark_as_output(y)
        with pytest.raises(RuntimeError):
            dr.score(y)
        dr.prepare(g)
        f = np.ones((2, nin, 1, 1), np.float32)
        dr.feed_data(x, f)
        dr.apply(g)
        with pytest.raises(RuntimeError):
            dr.score(h)
        with pytest.raises(ValueError):
            dr.score(y, k=21)
        with pytest.raises(TypeError):
            dr.score(y, labels=[0.5, 1.0])
        with pytest.raises(TypeError):
            dr.score(y, labels=[1, 2, 3])
        with pytest.raises(RuntimeError):
            dr.score(y, scale=-1.0)
        lp, ent, top, idx = dr.score(y, labels=[nout, -7], k=3)      # none of the classes; none given
        assert math.isnan(lp[0]) and lp[1] == 0.0 and np.isfinite(ent).all() and (np.diff(top, axis=1) <= 0).all()
        assert dr.lib.dR_scoreNode(g.ptr, h.ptr, 1.0, None, 0, None, None, 0, None, None) == 0
        dr.apply(g)                                                  # a refused call leaves the graph usable
