"""The operators at the answering end of a network: the fully connected layer with its weights in 8-bit floating point
(a scale for each block of 128), and the scoring of its outputs (log probabilities of given classes or tokens, entropy,
top alternatives).  One pass of each, in plain torch and through the library.

Fully connected, `n` rows of `nin` values to `nout` outputs.  Weights are e4m3 codes [nout][nin] with one float scale for
each 128 x 128 block.  Each row of the input is cut into blocks of 128 values; with A = max(largest |x| of the block,
2^-96) a value x becomes the e4m3 code q nearest (ties to even) to x * (448 / A) and stands for q * (A / 448), the three
operations in 32 bits.  out = act(bias + sum_k q(x)_k w_k), summed in 32 bits.

Log probabilities, `n` rows of `len` logits v at a temperature 1 / scale: lse = log sum exp(scale v); for every given label
scale v - lse (0 for a negative label: none given); entropy -sum p log p; the k largest logits as (log probability, index),
equal ones by ascending index.
"""
import math

import torch

own = False

BLOCK = 128
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
CODES = {"f32": 0, "bf16": 1, "f16": 2}


# ------------------------------------------------------------------------------------------------------------- the cases
def listed():
    fc = lambda name, n, nin, nout, dtype, out, act=0, bias=True: dict(  # noqa: E731
        name=name, op="fc", n=n, nin=nin, nout=nout, dtype=dtype, out=out, act=act, bias=bias)
    lp = lambda name, n, length, dtype, labels, k, scale=1.0, masked=0.0: dict(  # noqa: E731
        name=name, op="logprobs", n=n, len=length, dtype=dtype, labels=labels, k=k, scale=scale, masked=masked)
    return [
        # the classifier's hidden layer for one image: the smallest weight stream of the network's tail
        fc("fc_1x4096x4096_f32", 1, 4096, 4096, "f32", "f32", act=1),
        # the network's largest layer, one image at a time and a batch of 64
        fc("fc_1x25088x4096_f32", 1, 25088, 4096, "f32", "f32", act=1),
        fc("fc_64x25088x4096_f32", 64, 25088, 4096, "f32", "f32", act=1),
        # its last layer: class scores, no activation
        fc("fc_64x4096x1000_f32", 64, 4096, 1000, "f32", "f32"),
        # sizes that fit no tile
        fc("fc_37x1003x517_f16", 37, 1003, 517, "f16", "f16", act=1, bias=False),
        # a server's batch of rows, and a prompt or an offline run: bound by the products
        fc("fc_1000x4096x4096_bf16", 1000, 4096, 4096, "bf16", "bf16"),
        fc("fc_4096x8192x8192_bf16", 4096, 8192, 8192, "bf16", "bf16", bias=False),
        # the answer of a classifier with 1000 classes: one image, a batch
        lp("logprobs_1x1000_f32", 1, 1000, "f32", 1, 5),
        lp("logprobs_64x1000_f32", 64, 1000, "f32", 1, 5),
        # one generated token with its alternatives, at a temperature, over a large vocabulary with some of it forbidden
        lp("logprobs_1x131072_bf16", 1, 131072, "bf16", 1, 20, scale=1.25, masked=0.1),
        # a batch of sequences over an odd vocabulary
        lp("logprobs_77x50001_f16", 77, 50001, "f16", 2, 10),
        # scoring every position of a long text
        lp("logprobs_2048x131072_f32", 2048, 131072, "f32", 1, 20),
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    dtype = rng.choice(["f32", "bf16", "f16"])
    if rng.random() < 0.55:
        n, nin, nout = _log(rng, 1, 4096), _log(rng, 16, 25088), _log(rng, 8, 16384)
        if rng.random() < 0.5:  # layers whose widths are whole blocks, as most are
            nin, nout = -(-nin // BLOCK) * BLOCK, -(-nout // BLOCK) * BLOCK
        n = max(1, min(n, (4096 * 8192 * 8192) // (nin * nout)))
        return dict(op="fc", n=n, nin=nin, nout=nout, dtype=dtype, out=rng.choice([dtype, "f32"]),
                    act=rng.choice([0, 1]), bias=rng.random() < 0.5)
    n, length = _log(rng, 1, 2048), _log(rng, 2, 131072)
    return dict(op="logprobs", n=n, len=length, dtype=dtype, labels=rng.randint(1, 4), k=rng.randint(1, min(32, length)),
                scale=rng.choice([1.0, 1.0, 0.5, 1.25]), masked=rng.choice([0.0, 0.0, 0.1]))


def work(case):
    size = {"f32": 4, "bf16": 2, "f16": 2}
    n = case["n"]
    if case["op"] == "fc":
        nin, nout = case["nin"], case["nout"]
        scales = -(-nin // BLOCK) * -(-nout // BLOCK)
        moved = n * nin * size[case["dtype"]] + nin * nout + 4 * scales + (4 * nout if case["bias"] else 0)
        return {"bytes": moved + n * nout * size[case["out"]], "flops": 2 * n * nin * nout}
    # per logit: scale, subtract, exp, two sums, one comparison
    return {"bytes": n * case["len"] * size[case["dtype"]] + n * (8 * case["labels"] + 8 * case["k"] + 4), "flops": 6 * n * case["len"]}


# ------------------------------------------------------------------------------------------------------------ the inputs
def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    n = case["n"]
    if case["op"] == "fc":
        nin, nout = case["nin"], case["nout"]
        # activations behind a ReLU or a norm: rows of different sizes, a few channels larger than the others
        x = normal(n, nin) * (0.5 + torch.rand(n, 1, device="cuda", generator=g))
        x *= 1 + 7 * (torch.rand(nin, device="cuda", generator=g) < 0.01)
        if case["act"]:
            x = x.clamp_min(0)
        w = normal(nout, nin) * (2.0 / nin) ** 0.5
        kb, ob = -(-nin // BLOCK), -(-nout // BLOCK)
        p = torch.zeros(ob * BLOCK, kb * BLOCK, device="cuda")
        p[:nout, :nin] = w
        p = p.view(ob, BLOCK, kb, BLOCK)
        scales = p.abs().amax((1, 3)) / 448
        codes = (p / scales[:, None, :, None]).view(ob * BLOCK, kb * BLOCK)[:nout, :nin].to(torch.float8_e4m3fn).contiguous()
        return {"x": x.to(TYPES[case["dtype"]]), "codes": codes, "scales": scales, "bias": normal(nout) if case["bias"] else None}
    v = normal(n, case["len"]) * 2.5
    if case["masked"]:
        v.masked_fill_(torch.rand(v.shape, device="cuda", generator=g) < case["masked"], -math.inf)
        v[:, 0] = 0.5  # something is always allowed
    labels = torch.randint(0, case["len"], (n, case["labels"]), device="cuda", generator=g, dtype=torch.int32)
    labels[torch.rand(labels.shape, device="cuda", generator=g) < 0.05] = -1
    return {"logits": v.to(TYPES[case["dtype"]]), "labels": labels}


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if own:
        import deepracin_b200 as dr
        s["lib"] = dr.lib
        new = lambda *size, dtype=torch.float32: torch.empty(*size, dtype=dtype, device="cuda")  # noqa: E731
        stream = torch.cuda.current_stream().cuda_stream
        n = case["n"]
        if case["op"] == "fc":
            nin, nout = case["nin"], case["nout"]
            s["out"] = new(n, nout, dtype=TYPES[case["out"]])
            s["packed"] = new(dr.lib.dRk_fp8_fc_packed_bytes(nin, nout), dtype=torch.uint8)
            s["scratch"] = new(dr.lib.dRk_fp8_fc_scratch_bytes(n, nin, nout), dtype=torch.uint8)
            s["status"] = torch.zeros(1, dtype=torch.int32, device="cuda")
            if dr.lib.dRk_fp8_fc_pack_codes(stream, s["codes"].data_ptr(), nin, s["scales"].data_ptr(), s["packed"].data_ptr(), nin, nout):
                raise RuntimeError("dRk_fp8_fc_pack_codes refused %r" % (case,))
            plan = dr.lib.dRk_fp8_fc_plan(s["x"].data_ptr(), CODES[case["dtype"]], nin, s["packed"].data_ptr(),
                                          s["bias"].data_ptr() if case["bias"] else None, s["out"].data_ptr(), CODES[case["out"]], nout,
                                          s["scratch"].data_ptr(), n, nin, nout, case["act"], s["status"].data_ptr())
            if not plan:
                raise RuntimeError("dRk_fp8_fc_plan refused %r" % (case,))
            s["plan"] = Plan(dr.lib, plan)
        else:
            s["logprob"], s["entropy"] = new(n, case["labels"]), new(n)
            s["top"], s["index"] = new(n, case["k"]), new(n, case["k"], dtype=torch.int32)
    return s


class Plan:
    """A layer's plan, freed with the state that holds it."""

    def __init__(self, lib, pointer):
        self.lib, self.pointer = lib, pointer

    def __del__(self):
        self.lib.dRk_fp8_fc_free(self.pointer)


# -------------------------------------------------------------------------------------------------------------- one pass
def run(state):
    case = state["case"]
    if own:
        lib, stream = state["lib"], torch.cuda.current_stream().cuda_stream
        if case["op"] == "fc":
            if lib.dRk_fp8_fc_run(stream, state["plan"].pointer):
                raise RuntimeError("dRk_fp8_fc_run failed")
            return state["out"]
        logits = state["logits"]
        if lib.dRk_logprobs(stream, logits.data_ptr(), CODES[case["dtype"]], case["len"], case["n"], case["len"], case["scale"],
                            state["labels"].data_ptr(), case["labels"], state["logprob"].data_ptr(), state["entropy"].data_ptr(),
                            case["k"], state["top"].data_ptr(), state["index"].data_ptr()):
            raise RuntimeError("dRk_logprobs failed")
        return [state["logprob"], state["entropy"], state["top"], state["index"]]
    return plain_fc(state) if case["op"] == "fc" else plain_logprobs(state)


def plain_fc(state):
    case, x, codes, scales = state["case"], state["x"].float(), state["codes"], state["scales"]
    n, nin, nout = case["n"], case["nin"], case["nout"]
    kb = scales.shape[1]
    blocks = torch.nn.functional.pad(x, (0, kb * BLOCK - nin)).view(n, kb, BLOCK)
    largest = blocks.abs().amax(2, keepdim=True).clamp_min(2.0 ** -96)
    top = torch.full((), 448.0, device=x.device)  # a tensor: torch divides by or into a plain number through a reciprocal
    q = (blocks * (top / largest)).to(torch.float8_e4m3fn).float() * (largest / top)
    spread = scales.repeat_interleave(BLOCK, 0)[:nout].repeat_interleave(BLOCK, 1)[:, :nin]
    out = q.view(n, kb * BLOCK)[:, :nin] @ (codes.float() * spread).t()
    if case["bias"]:
        out = out + state["bias"]
    if case["act"]:
        out = out.clamp_min(0)
    return out.to(TYPES[case["out"]])


def plain_logprobs(state):
    case, logits, labels = state["case"], state["logits"], state["labels"].long()
    v = logits.float() * case["scale"]
    d = v - v.amax(1, keepdim=True)
    e = torch.exp(d)
    total = e.sum(1, keepdim=True, dtype=torch.float64)
    log_total = torch.log(total)
    entropy = log_total[:, 0] - torch.where(e > 0, e * d, 0.0).sum(1, dtype=torch.float64) / total[:, 0]
    given = torch.where(labels >= 0, (d.gather(1, labels.clamp_min(0)) - log_total), 0.0)
    # order by value and then by ascending index: a whole number that holds both
    bits = logits.float().view(torch.int32)
    bits = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long()
    column = torch.arange(case["len"], device=logits.device)
    index = (bits * 2 ** 32 + (2 ** 31 - column)).topk(case["k"], dim=1).indices
    top = d.gather(1, index) - log_total
    return [given.float(), entropy.float(), top.float(), index.int()]


# ------------------------------------------------------------------------------------------------- the definition, 64 bits
def _nearest_e4m3(v):
    """The e4m3 value nearest to v, ties to even: 3 bits behind the leading one, exponents from -6 on, at most 448."""
    exponent = (torch.frexp(v)[1] - 1).clamp_min(-6)
    step = torch.ldexp(torch.ones_like(v), exponent - 3)
    return (torch.round(v / step) * step).clamp(-448, 448)


def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "fc":
        x = s["x"].double()
        w = s["codes"].double()
        out = torch.zeros(case["n"], case["nout"], dtype=torch.float64, device="cuda")
        top = torch.full((), 448.0, dtype=torch.float64, device="cuda")
        for b in range(s["scales"].shape[1]):
            xb, wb = x[:, b * BLOCK:(b + 1) * BLOCK], w[:, b * BLOCK:(b + 1) * BLOCK]
            largest = xb.abs().amax(1, keepdim=True).clamp_min(2.0 ** -96)
            # the factors and the product are rounded to 32 bits by the definition
            scaled = (xb * (top / largest).float().double()).float().double()
            part = _nearest_e4m3(scaled) @ wb.t()
            rows = torch.arange(case["nout"], device="cuda") // BLOCK
            out += part * (largest / top).float().double() * s["scales"][rows, b].double()
        if case["bias"]:
            out += s["bias"].double()
        return out.clamp_min(0) if case["act"] else out
    scale = torch.tensor(case["scale"], dtype=torch.float32).double().item()
    logits, n = s["logits"], case["n"]
    given = torch.zeros(n, case["labels"], dtype=torch.float64, device="cuda")
    entropy = torch.zeros(n, dtype=torch.float64, device="cuda")
    top = torch.zeros(n, case["k"], dtype=torch.float64, device="cuda")
    for first in range(0, n, 128):
        rows = slice(first, min(n, first + 128))
        v = logits[rows].double() * scale
        lse = torch.logsumexp(v, 1, keepdim=True)
        logp = v - lse
        entropy[rows] = -torch.where(logp > -math.inf, logp.exp() * logp, 0.0).sum(1)
        labels = s["labels"][rows].long()
        given[rows] = torch.where(labels >= 0, logp.gather(1, labels.clamp_min(0)), 0.0)
        top[rows] = logp.sort(1, descending=True).values[:, :case["k"]]
    return [given, entropy, top, None]
