"""GPU tests of the 8-bit fully connected layer (dRk_fp8_fc_*) against its definition in 64 bits.

The codes and scales are fixed by the definition (32-bit operations, nearest even), so the reference uses the same ones and the
kernel may differ by the rounding of its 32-bit sums alone: a sum of the products of nin pairs, taken as blocks of 128 whose
partial sums are scaled and added, passes at most 128 + blocks + 8 roundings (the 8: the scale product, its application, bias
and output), each at most one step 2^-23 of the magnitudes summed (truncation included; rounding would be half of it).
Outputs in 16 bits add half a step of their own type."""
import ctypes

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

TYPES = {0: torch.float32, 1: torch.bfloat16, 2: torch.float16}
F32, BF16, F16 = 0, 1, 2


def _lib():
    import deepracin_b200 as dr
    return dr.lib


def nearest_e4m3(v):
    """e4m3 value nearest to v (float64), ties to even; NaN passes"""
    e = (torch.frexp(v)[1] - 1).clamp_min(-6)
    step = torch.ldexp(torch.ones_like(v), e - 3)
    return (torch.round(v / step) * step).clamp(-448, 448)


def quantized(x):
    """values that the rows of x stand for after rounding, float64"""
    n, nin = x.shape
    kb = -(-nin // 128)
    b = torch.zeros(n, kb * 128, dtype=torch.float32, device=x.device)
    b[:, :nin] = x.float()
    b = b.view(n, kb, 128)
    top = torch.full((), 448.0, device=x.device)
    a = b.abs().amax(2, keepdim=True).clamp_min(2.0 ** -96)
    q = nearest_e4m3((b * (top / a)).double())
    return (q * (a / top).double()).view(n, kb * 128)[:, :nin]


def make_weights(nin, nout, seed):
    g = torch.Generator().manual_seed(seed)
    kb, ob = -(-nin // 128), -(-nout // 128)
    codes = torch.randint(0, 256, (nout, nin), generator=g, dtype=torch.uint8)
    codes[(codes & 0x7f) == 0x7f] = 0x38      # no NaN codes
    scales = torch.rand(ob, kb, generator=g) * 0.01 + 1e-4
    return codes.cuda(), scales.cuda()


def dequantized(codes, scales):
    nout, nin = codes.shape
    w = codes.view(torch.float8_e4m3fn).double()
    s = scales.double().repeat_interleave(128, 0)[:nout].repeat_interleave(128, 1)[:, :nin]
    return w * s


class Layer:
    def __init__(self, x, codes, scales, bias, out_type, act, in_type=F32, ldi=None, ldo=None, xptr=None, out=None):
        lib = _lib()
        self.lib = lib
        self.n, (self.nout, self.nin) = x.shape[0], codes.shape
        dev = x.device
        self.packed = torch.empty(lib.dRk_fp8_fc_packed_bytes(self.nin, self.nout), dtype=torch.uint8, device=dev)
        self.scratch = torch.empty(lib.dRk_fp8_fc_scratch_bytes(self.n, self.nin, self.nout), dtype=torch.uint8, device=dev)
        self.status = torch.zeros(1, dtype=torch.int32, device=dev)
        self.ldo = ldo or self.nout
        self.out = torch.full((self.n, self.ldo), -77.0, dtype=TYPES[out_type], device=dev) if out is None else out
        self.keep = (x, codes, scales, bias)
        stream = torch.cuda.current_stream(dev).cuda_stream
        assert lib.dRk_fp8_fc_pack_codes(stream, codes.data_ptr(), codes.stride(0), scales.data_ptr(), self.packed.data_ptr(), self.nin, self.nout) == 0
        self.plan = lib.dRk_fp8_fc_plan(x.data_ptr() if xptr is None else xptr, in_type, ldi or self.nin, self.packed.data_ptr(),
                                        bias.data_ptr() if bias is not None else None, self.out.data_ptr(), out_type, self.ldo,
                                        self.scratch.data_ptr(), self.n, self.nin, self.nout, act, self.status.data_ptr())
        assert self.plan

    def run(self, stream=None):
        st = torch.cuda.current_stream().cuda_stream if stream is None else stream
        assert self.lib.dRk_fp8_fc_run(st, self.plan) == 0

    def result(self):
        torch.cuda.synchronize()
        assert int(self.status.item()) == 0
        return self.out[:, :self.nout]

    def __del__(self):
        if getattr(self, "plan", None):
            self.lib.dRk_fp8_fc_free(self.plan)


def check(got, xq, w, bias, act, kb):
    ref, mag = xq @ w.t(), xq.abs() @ w.abs().t()
    if bias is not None:
        ref, mag = ref + bias.double(), mag + bias.double().abs()
    if act:
        ref = ref.clamp_min(0)
    bound = mag * (128 + kb + 8) * 2.0 ** -23 + ref.abs() * torch.finfo(got.dtype).eps / 2 + torch.finfo(got.dtype).tiny
    err = (got.double() - ref).abs()
    assert bool((err <= bound).all()), float((err / bound).max())


SHAPES = [(1, 1, 1), (1, 128, 128), (2, 129, 127), (3, 127, 257), (5, 16, 3), (16, 256, 384), (17, 1000, 100), (37, 1003, 517),
          (33, 2176, 1000), (64, 4096, 1000), (65, 640, 130), (96, 1500, 129), (128, 384, 256), (129, 300, 200), (200, 2049, 260),
          (256, 512, 512), (300, 1024, 640), (513, 256, 1000), (1000, 512, 300), (1, 25088, 384), (1030, 1290, 2060), (2500, 384, 515),
          # several tiles of 64 rows, in shares and whole
          (150, 8300, 300), (330, 5000, 1800), (70, 4100, 4500),
          # pairs of CTAs on 256 x 256 tiles: ragged edges, an odd number of weight blocks, one block, several tiles for each pair
          (129, 2000, 8200), (333, 3000, 4100), (1500, 1290, 2300), (2100, 900, 1100), (2500, 300, 8200), (3000, 100, 5000)]


@pytest.mark.parametrize("types", [(F32, F32), (BF16, BF16), (F16, F32), (F32, F16)])
@pytest.mark.parametrize("n,nin,nout", SHAPES)
def test_against_the_definition(n, nin, nout, types):
    tin, tout = types
    g = torch.Generator().manual_seed(n * 7 + nin + nout)
    x = (torch.randn(n, nin, generator=g) * (0.25 + torch.rand(n, 1, generator=g))).to(TYPES[tin]).cuda()
    codes, scales = make_weights(nin, nout, nin * 3 + nout)
    bias = torch.randn(nout, generator=g).cuda() if (n + nout) % 2 else None
    act = n % 2
    if tout == F16:
        scales = scales * 0.02      # keeps the outputs inside the range of 16 bits
    layer = Layer(x, codes, scales, bias, tout, act, tin)
    layer.run()
    check(layer.result(), quantized(x), dequantized(codes, scales), bias, act, -(-nin // 128))


@pytest.mark.parametrize("tout", [F32, BF16, F16])
@pytest.mark.parametrize("n,nin,nout,ldo", [(2501, 300, 8200, 8200), (2501, 300, 8200, 8204), (3001, 128, 5000, 5008), (2050, 257, 9001, 9001), (4001, 256, 256, 256), (900, 128, 1027, 1032)])
def test_bias_and_activation_of_many_tiles(n, nin, nout, ldo, tout):
    """several tiles for each pair of CTAs, whose bias is fetched a tile ahead; rows that can be stored 16 bytes at a time and others"""
    g = torch.Generator().manual_seed(n + ldo)
    x = torch.randn(n, nin, generator=g).cuda()
    codes, scales = make_weights(nin, nout, 21)
    scales = scales * 0.02
    bias = torch.randn(nout, generator=g).cuda()
    layer = Layer(x, codes, scales, bias, tout, 1, F32, ldo=ldo)
    layer.run()
    check(layer.result(), quantized(x), dequantized(codes, scales), bias, 1, -(-nin // 128))
    assert bool((layer.out[:, nout:] == -77.0).all())


@pytest.mark.parametrize("n,nin,nout", [(1, 700, 300), (37, 1003, 517), (300, 520, 389), (1100, 650, 1300), (1500, 1290, 2301)])
@pytest.mark.parametrize("tin,tout", [(F32, F32), (BF16, F16)])
def test_pitches_and_alignment(n, nin, nout, tin, tout):
    """rows further apart than they are long, starting off every vector boundary; what lies between the rows stays"""
    g = torch.Generator().manual_seed(n)
    ldi, ldo = nin + 5, nout + 3
    flat = torch.full((n * ldi + 1,), float("nan"), dtype=TYPES[tin], device="cuda")
    view = flat[1:].view(n, ldi)
    x = torch.randn(n, nin, generator=g).to(TYPES[tin]).cuda()
    view[:, :nin] = x
    codes, scales = make_weights(nin, nout, 5)
    if tout == F16:
        scales = scales * 0.02
    oflat = torch.full((n * ldo + 1,), -77.0, dtype=TYPES[tout], device="cuda")
    out = oflat[1:].view(n, ldo)
    layer = Layer(x, codes, scales, None, tout, 0, tin, ldi=ldi, ldo=ldo, xptr=view.data_ptr(), out=out)
    layer.run()
    check(layer.result(), quantized(x), dequantized(codes, scales), None, 0, -(-nin // 128))
    assert bool((out[:, nout:] == -77.0).all()) and float(oflat[0]) == -77.0


@pytest.mark.parametrize("n,nin,ldi", [(700, 4099, 4099), (2600, 1025, 1027), (1200, 2050, 2051)])
def test_many_rows_off_every_boundary(n, nin, ldi):
    g = torch.Generator().manual_seed(nin)
    flat = torch.full((n * ldi + 1,), float("nan"), device="cuda")
    view = flat[1:].view(n, ldi)
    x = (torch.randn(n, nin, generator=g) * (0.25 + torch.rand(n, 1, generator=g))).cuda()
    x[5] = 0
    view[:, :nin] = x
    codes, scales = make_weights(nin, 130, 8)
    layer = Layer(x, codes, scales, None, F32, 0, F32, ldi=ldi, xptr=view.data_ptr())
    layer.run()
    check(layer.result(), quantized(x), dequantized(codes, scales), None, 0, -(-nin // 128))


def test_codes_with_a_row_pitch_and_packing_of_the_float_matrix():
    lib = _lib()
    nin, nout = 333, 259
    g = torch.Generator().manual_seed(3)
    w = torch.randn(nin, nout, generator=g).cuda()
    w[:128, 128:256] = 0            # a block of zeros
    packed = torch.empty(lib.dRk_fp8_fc_packed_bytes(nin, nout), dtype=torch.uint8, device="cuda")
    back = torch.empty_like(w)
    st = torch.cuda.current_stream().cuda_stream
    assert lib.dRk_fp8_fc_pack_weights(st, w.data_ptr(), packed.data_ptr(), nin, nout) == 0
    assert lib.dRk_fp8_fc_unpack_weights(st, packed.data_ptr(), back.data_ptr(), nin, nout) == 0
    kb, ob = -(-nin // 128), -(-nout // 128)
    p = torch.zeros(kb * 128, ob * 128, device="cuda")
    p[:nin, :nout] = w
    p = p.view(kb, 128, ob, 128)
    a = p.abs().amax((1, 3), keepdim=True).clamp_min(2.0 ** -96)
    top = torch.full((), 448.0, device="cuda")
    want = (nearest_e4m3((p * (top / a)).double()) * (a / top).double()).float().view(kb * 128, ob * 128)[:nin, :nout]
    assert torch.equal(back, want)
    # the same codes brought in with a row pitch give the same packed bytes
    codes = nearest_e4m3((p * (top / a)).double()).float().view(kb * 128, ob * 128)[:nin, :nout].t().contiguous().to(torch.float8_e4m3fn).view(torch.uint8)
    wide = torch.full((nout, nin + 9), 0x7f, dtype=torch.uint8, device="cuda")
    wide[:, :nin] = codes
    scales = (a / top).view(kb, ob).t().contiguous()
    again = torch.empty_like(packed)
    assert lib.dRk_fp8_fc_pack_codes(st, wide.data_ptr(), nin + 9, scales.data_ptr(), again.data_ptr(), nin, nout) == 0
    torch.cuda.synchronize()
    # -0 and +0 are the same value; everything else is the same byte
    zero = (packed[:kb * ob * 16384] & 0x7f) == 0
    same = packed[:kb * ob * 16384] == again[:kb * ob * 16384]
    assert bool((same | (zero & ((again[:kb * ob * 16384] & 0x7f) == 0))).all())
    assert torch.equal(packed[kb * ob * 16384:].view(torch.float32), again[kb * ob * 16384:].view(torch.float32))


@pytest.mark.parametrize("n,nin,nout", [(4, 384, 200), (40, 384, 200), (700, 384, 400), (2100, 1408, 1100)])
def test_rows_of_zeros_infinities_and_nan(n, nin, nout):
    g = torch.Generator().manual_seed(n)
    x = torch.randn(n, nin, generator=g).cuda()
    x[0] = 0
    x[1, 130] = float("inf")
    x[2, 5] = float("nan")
    x[3] *= 1e-38                   # below the smallest scale: codes of almost nothing, no infinities
    codes, scales = make_weights(nin, nout, 1)
    codes[codes == 0] = 0x10        # a zero weight would turn inf * 0 into NaN as well; the row is NaN either way
    layer = Layer(x, codes, scales, None, F32, 0)
    layer.run()
    got = layer.result()
    assert bool((got[0] == 0).all())
    assert bool(got[1].isnan().all()) and bool(got[2].isnan().all())
    fine = torch.tensor([0] + list(range(3, n)), device="cuda")
    check(got[fine], quantized(x[fine]), dequantized(codes, scales), None, 0, nin // 128)
    relu = Layer(x, codes, scales, None, F32, 1)
    relu.run()
    assert bool(relu.result()[2].isnan().all())


def test_nan_weights_stay_in_their_column():
    codes, scales = make_weights(300, 200, 1)
    codes[7, 299] = 0x7f
    x = torch.randn(5, 300, device="cuda")
    layer = Layer(x, codes, scales, None, F32, 0)
    layer.run()
    nan = layer.result().isnan()
    assert bool(nan[:, 7].all()) and int(nan.sum()) == 5


def test_same_answer_every_time_and_after_other_work():
    for n, nin, nout in [(1, 4096, 512), (50, 2048, 512), (600, 1024, 512), (2100, 1024, 1100)]:
        codes, scales = make_weights(nin, nout, 2)
        x = torch.randn(n, nin, device="cuda")
        layer = Layer(x, codes, scales, None, F32, 0)
        layer.run()
        first = layer.result().clone()
        other = Layer(torch.randn(77, 513, device="cuda"), *make_weights(513, 99, 4), None, F32, 0)
        for _ in range(5):
            other.run()
            layer.run()
        assert torch.equal(first, layer.result())


def test_streams_and_graph_capture():
    """two plans at once on two streams; a plan captured, replayed on new inputs; a plan on a stream other than torch's"""
    shapes = [(1, 4096, 1000), (64, 2048, 640), (520, 1024, 700), (2100, 1024, 1100)]
    for n, nin, nout in shapes:
        codes, scales = make_weights(nin, nout, 9)
        w = dequantized(codes, scales)
        x1, x2 = torch.randn(n, nin, device="cuda"), torch.randn(n, nin, device="cuda")
        a, b = Layer(x1, codes, scales, None, F32, 0), Layer(x2, codes, scales, None, F32, 0)
        s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
        torch.cuda.synchronize()
        for _ in range(10):
            a.run(s1.cuda_stream)
            b.run(s2.cuda_stream)
        check(a.result(), quantized(x1), w, None, 0, nin // 128)
        check(b.result(), quantized(x2), w, None, 0, nin // 128)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s1):
            a.run(s1.cuda_stream)
        for _ in range(3):
            x1.copy_(torch.randn(n, nin, device="cuda"))
            a.out.fill_(float("nan"))
            torch.cuda.synchronize()
            graph.replay()
            check(a.result(), quantized(x1), w, None, 0, nin // 128)
        del graph


def test_weights_packed_just_before_the_run():
    """the layer's weights may be written by the launch in front of it on the same stream"""
    lib = _lib()
    n, nin, nout = 8, 8192, 512
    x = torch.randn(n, nin, device="cuda")
    codes, scales = make_weights(nin, nout, 1)
    layer = Layer(x, codes, scales, None, F32, 0)
    for seed in range(4):
        codes, scales = make_weights(nin, nout, 10 + seed)
        torch.cuda.synchronize()
        st = torch.cuda.current_stream().cuda_stream
        assert lib.dRk_fp8_fc_pack_codes(st, codes.data_ptr(), nin, scales.data_ptr(), layer.packed.data_ptr(), nin, nout) == 0
        layer.run()
        check(layer.result(), quantized(x), dequantized(codes, scales), None, 0, nin // 128)


def test_run_refuses_a_stream_of_another_device():
    if torch.cuda.device_count() < 2:
        pytest.skip("one device")
    layer = Layer(torch.randn(2, 128, device="cuda:0"), *make_weights(128, 16, 1), None, F32, 0)
    other = torch.cuda.Stream(device=1)
    assert layer.lib.dRk_fp8_fc_run(other.cuda_stream, layer.plan) == -6
