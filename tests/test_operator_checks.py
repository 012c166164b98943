"""Refusals of the operator entry points, on the host: every call here is refused before anything is launched."""
import ctypes

import numpy as np
import pytest

import deepracin_b200 as dr

lib = dr.lib
P = 1 << 20         # a non-null, aligned address that is never read


def fc_plan(**kw):
    a = dict(inp=P, in_type=0, ldi=256, packed=P, bias=P, out=P, out_type=0, ldo=128, scratch=P, n=4, nin=256, nout=128, act=0, status=None)
    a.update(kw)
    return lib.dRk_fp8_fc_plan(a["inp"], a["in_type"], a["ldi"], a["packed"], a["bias"], a["out"], a["out_type"], a["ldo"], a["scratch"],
                               a["n"], a["nin"], a["nout"], a["act"], a["status"])


@pytest.mark.parametrize("change,says", [
    (dict(inp=None), "null pointer"), (dict(packed=None), "null pointer"), (dict(out=None), "null pointer"), (dict(scratch=None), "null pointer"),
    (dict(in_type=3), "unknown element type"), (dict(out_type=-1), "unknown element type"),
    (dict(n=0), "sizes outside"), (dict(nin=0), "sizes outside"), (dict(nout=-5), "sizes outside"),
    (dict(n=2 ** 31 - 1, nin=2 ** 20, ldi=2 ** 20), "sizes outside"), (dict(nin=2 ** 31 - 1, nout=2 ** 31 - 1, ldi=2 ** 31, ldo=2 ** 31), "sizes outside"),
    (dict(ldi=255), "rows overlap"), (dict(ldo=127), "rows overlap"), (dict(n=1, ldi=-1), "negative"),
    (dict(act=2), "activation"), (dict(inp=P + 2), "not aligned to its element"), (dict(out=P + 1), "not aligned to its element"),
    (dict(in_type=1, inp=P + 1), "not aligned to its element"), (dict(bias=P + 2), "not aligned to its element"),
    (dict(packed=P + 8), "16-byte"), (dict(scratch=P + 4), "16-byte")])
def test_fp8_fc_plan_refuses(change, says, capfd):
    assert not fc_plan(**change)
    err = capfd.readouterr().err
    assert err.startswith("dRk_fp8_fc_plan: ") and says in err


def test_fp8_fc_sizes():
    assert lib.dRk_fp8_fc_packed_bytes(128, 128) == 16384 + 4
    assert lib.dRk_fp8_fc_packed_bytes(129, 1) == 2 * (16384 + 4)
    assert lib.dRk_fp8_fc_packed_bytes(0, 5) == 0 and lib.dRk_fp8_fc_scratch_bytes(0, 5, 5) == 0
    assert lib.dRk_fp8_fc_scratch_bytes(3, 300, 10) >= 3 * 3 * (128 + 4)
    assert lib.dRk_fp8_fc_supported(1, 1, 1) == 1 and lib.dRk_fp8_fc_supported(4096, 25088, 16384) == 1


def test_fp8_fc_packing_and_run_refuse(capfd):
    assert lib.dRk_fp8_fc_pack_weights(None, None, P, 128, 128) == -1
    assert lib.dRk_fp8_fc_pack_weights(None, P, P + 1, 128, 128) == -1
    assert lib.dRk_fp8_fc_pack_weights(None, P, P, 0, 128) == -1
    assert lib.dRk_fp8_fc_pack_codes(None, P, 127, P, P, 128, 128) == -1
    assert lib.dRk_fp8_fc_pack_codes(None, P, 128, None, P, 128, 128) == -1
    assert lib.dRk_fp8_fc_unpack_weights(None, P, None, 128, 128) == -1
    assert lib.dRk_fp8_fc_run(None, None) == -1
    lib.dRk_fp8_fc_free(None)
    err = capfd.readouterr().err
    assert "rows of codes overlap" in err and "dRk_fp8_fc_run: no plan" in err


def logprobs(**kw):
    a = dict(logits=P, type=0, ld=100, n=2, length=100, scale=1.0, labels=P, m=1, logprob=P, entropy=P, k=5, top=P, index=P)
    a.update(kw)
    return lib.dRk_logprobs(None, a["logits"], a["type"], a["ld"], a["n"], a["length"], a["scale"], a["labels"], a["m"], a["logprob"], a["entropy"],
                            a["k"], a["top"], a["index"])


@pytest.mark.parametrize("change,says", [
    (dict(type=5), "unknown element type"), (dict(n=0), "at least one row"), (dict(length=0), "at least one row"), (dict(n=-1), "at least one row"),
    (dict(ld=99), "rows overlap"), (dict(m=-1), "number of labels"), (dict(k=33), "number of labels"), (dict(k=-1), "number of labels"),
    (dict(length=4, ld=4, k=5), "number of labels"), (dict(logits=None), "null pointer"), (dict(labels=None), "null pointer"),
    (dict(logprob=None), "null pointer"), (dict(top=None), "null pointer"), (dict(index=None), "null pointer"),
    (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"), (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"), (dict(scale=3e38), "scale"),
    (dict(logits=P + 2), "not aligned"), (dict(type=2, logits=P + 1), "not aligned"), (dict(labels=P + 1), "not aligned"), (dict(entropy=P + 2), "not aligned")])
def test_logprobs_refuses(change, says, capfd):
    assert logprobs(**change) == -1
    err = capfd.readouterr().err
    assert err.startswith("dRk_logprobs: ") and says in err


def dry_graph(batch, fp8, dims=(300, 200, 40)):
    env = dr.Environment().__enter__()
    g = env.create_graph("CHW")
    x = dr.feed_node(g, [dims[0], 1, 1])
    node = x
    for nin, nout in zip(dims, dims[1:]):
        node = dr.Fully_Connected(node, [nin, nout], "relu", np.zeros((nin, nout), np.float32), np.zeros(nout, np.float32))
    dr.mark_as_output(node)
    lib.dR_setBatchSize(g.ptr, batch)
    assert lib.dR_setFp8FullyConnected(g.ptr, fp8)
    lib.dR_config(g.ptr, b"", 1, 0, 0, 0, b"")
    lib.dR_setDryRun(g.ptr, 1)
    assert lib.dR_prepare(g.ptr)
    return env, g, node


def test_graph_with_8_bit_layers_plans_its_scratch():
    env, g, _ = dry_graph(7, 1)
    need = max(lib.dRk_fp8_fc_scratch_bytes(7, 300, 200), lib.dRk_fp8_fc_scratch_bytes(7, 200, 40))
    assert lib.dR_getScratchFloats(g.ptr) == (need + 3) // 4
    assert not lib.dR_setFp8FullyConnected(g.ptr, 0)        # too late
    env.__exit__(None, None, None)
    env, g, _ = dry_graph(7, 0)
    assert lib.dR_getScratchFloats(g.ptr) != (need + 3) // 4
    env.__exit__(None, None, None)


def test_score_node_refuses_without_a_device(capfd):
    env, g, node = dry_graph(2, 0)
    assert not lib.dR_scoreNode(g.ptr, node.ptr, 1.0, None, 0, None, P, 0, None, None)
    env.__exit__(None, None, None)
    with dr.Environment() as env:
        g = env.create_graph("CHW")
        x = dr.feed_node(g, [4, 1, 1])
        assert not lib.dR_scoreNode(g.ptr, x.ptr, 1.0, None, 0, None, P, 0, None, None)
