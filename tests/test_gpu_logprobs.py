"""GPU tests of dRk_logprobs against its definition in 64 bits.

Tolerances: with d = scale (v - max), rounding v - max and its product with the scale moves d by at most 2 * 2^-24 |d|, which
moves e = exp(d) by as much, relatively, on top of 2^-22 of the exponential itself; a sum of len positive terms in 32 bits is
off by at most 2^-24 for each of the additions a term passes, at most len / 128 + 64 (at least 128 partial sums run side by
side).  The indices have to be equal."""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]


def call(v, labels=None, k=0, scale=1.0, ld=None, want_entropy=True, n=None, length=None, ptr=None, stream=None, outs=None):
    import deepracin_b200 as dr
    n, length = n or v.shape[0], length or v.shape[1]
    m = 0 if labels is None else labels.shape[1]
    lp, h, top, idx = outs or (torch.full((n, m), 9.0, device="cuda"), torch.full((n,), 9.0, device="cuda"), torch.full((n, k), 9.0, device="cuda"),
                               torch.full((n, k), -9, dtype=torch.int32, device="cuda"))
    st = torch.cuda.current_stream().cuda_stream if stream is None else stream
    rc = dr.lib.dRk_logprobs(st, ptr or v.data_ptr(), TYPES.index(v.dtype), ld or length, n, length, scale, labels.data_ptr() if m else None, m,
                             lp.data_ptr() if m else None, h.data_ptr() if want_entropy else None, k, top.data_ptr() if k else None, idx.data_ptr() if k else None)
    assert rc == 0
    return lp, h, top, idx


def order(v, k):
    """indices of the k largest, ties by ascending index, NaN first"""
    x = torch.where(v.isnan(), math.inf, v.double())
    first = torch.sort((~v.isnan()).int(), dim=1, stable=True).indices      # NaN to the front, otherwise as they stand
    x = x.gather(1, first)
    nan = v.isnan().gather(1, first)
    by = torch.sort(x, dim=1, descending=True, stable=True).indices
    # an infinity ties with the NaN placeholders but stands behind them already
    del nan
    return first.gather(1, by)[:, :k].int()


def check(v, got, labels, k, scale):
    lp, h, top, idx = [t.cpu() for t in got]
    v = v.detach().cpu()
    n, length = v.shape
    s = float(torch.tensor(scale, dtype=torch.float32))
    x = v.double() * s
    mx = x.amax(1, keepdim=True)
    none = (v == -math.inf).all(1)
    bad = v.isnan().any(1) | (v == math.inf).any(1)
    d = torch.where(none[:, None], -math.inf, x - mx)
    S = torch.where(none, 1.0, d.exp().sum(1))
    logS = S.log()[:, None]
    p = d.exp() / S[:, None]
    fin = torch.where(p > 0, d, 0.0)
    mean, sq = (p * fin).sum(1), (p * fin * fin).sum(1)
    H = torch.where(none, 0.0, logS[:, 0] - mean)
    chain = (length / 128 + 64) * 2.0 ** -24
    sum_err = chain + 2.0 ** -22 + 2.0 ** -23 * mean.abs()
    fine = ~bad
    h_err = 2 * sum_err * (1 + mean.abs()) + 2.0 ** -22 * (sq + logS[:, 0].abs() + mean.abs())
    assert bool(((h.double() - H).abs() <= h_err)[fine].all()), float(((h.double() - H).abs() / h_err)[fine].max())
    assert bool(h[bad].isnan().all())
    logp = d - logS

    def close(got, want, dd, rows):
        # the outputs are held in 32 bits: what lies beyond their range (2^128 less half a step) rounds to an infinity
        want = torch.where(want.abs() >= 2.0 ** 128 - 2.0 ** 103, torch.sign(want) * math.inf, want)
        err = (got.double() - want).abs()
        tol = sum_err[:, None] + 2.0 ** -22 * (torch.where(dd.isfinite(), dd, 0.0).abs() + logS.abs())
        good = torch.where(want.isfinite(), err <= tol, got.double() == want)
        assert bool(good[rows].all())

    if k:
        want = order(v, k)
        assert torch.equal(idx, want)
        close(top, logp.gather(1, want.long()), d.gather(1, want.long()), fine)
        assert bool(top[bad].isnan().all())
    if labels is not None:
        lab = labels.cpu().long()
        inside = (lab >= 0) & (lab < length)
        at = lab.clamp(0, length - 1)
        assert bool((lp[lab < 0] == 0).all()) and bool(lp[lab >= length].isnan().all())
        w = torch.where(inside, logp.gather(1, at), 0.0)
        g = torch.where(inside, lp, 0.0)
        close(g, w, torch.where(inside, d.gather(1, at), 0.0), fine)
        assert bool(lp[bad][inside[bad]].isnan().all())


LENS = [1, 2, 3, 7, 31, 32, 33, 100, 1000, 1023, 4097, 8192, 50001, 131075]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("length", LENS)
def test_against_the_definition(length, dtype):
    g = torch.Generator().manual_seed(length)
    for n, k, m, scale in [(1, min(5, length), 1, 1.0), (3, min(32, length), 4, 1.25), (40, min(20, length), 0, 0.5), (2, 0, 2, 1.0)]:
        v = (torch.randn(n, length, generator=g) * 2.5).to(dtype).cuda()
        labels = torch.randint(0, length, (n, m), generator=g, dtype=torch.int32).cuda() if m else None
        check(v, call(v, labels, k, scale), labels, k, scale)


@pytest.mark.parametrize("n,length", [(147, 999), (148, 1000), (149, 4000), (295, 3001), (300, 700), (600, 5000), (3000, 130)])
def test_many_rows(n, length):
    v = torch.randn(n, length, device="cuda") * 3
    labels = torch.randint(0, length, (n, 1), device="cuda", dtype=torch.int32)
    check(v, call(v, labels, 7), labels, 7, 1.0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,length,pad", [(3, 1000, 1), (5, 4099, 3), (2, 60000, 5), (400, 517, 2)])
def test_pitch_and_alignment(n, length, pad, dtype):
    ld = length + pad
    flat = torch.full((n * ld + 1,), float("nan"), dtype=dtype, device="cuda")
    view = flat[1:].view(n, ld)
    v = torch.randn(n, length, device="cuda").to(dtype)
    view[:, :length] = v
    check(v, call(v, None, 9, 1.0, ld=ld, ptr=view.data_ptr()), None, 9, 1.0)


@pytest.mark.parametrize("length", [40, 1000, 33000, 131072])
@pytest.mark.parametrize("kind", ["equal", "three values", "ascending", "descending", "one stripe", "zeros of both signs", "blocks"])
def test_orders_that_are_hard_for_a_selection(kind, length):
    n, k = 3, 32
    i = torch.arange(length, device="cuda")
    if kind == "equal":
        v = torch.full((n, length), 1.5, device="cuda")
    elif kind == "three values":
        v = torch.randint(0, 3, (n, length), device="cuda").float()
    elif kind == "ascending":
        v = (i.float() / 64).expand(n, length).contiguous()
    elif kind == "descending":
        v = (-i.float() / 64).expand(n, length).contiguous()
    elif kind == "one stripe":      # the largest all sit at one distance from one another
        v = torch.randn(n, length, device="cuda")
        v[:, 5::512] += 50
        v[:, 2::2048] += 100
    elif kind == "zeros of both signs":
        v = torch.where(torch.randint(0, 2, (n, length), device="cuda") == 1, 0.0, -0.0)
    else:                           # the largest all sit side by side
        v = torch.randn(n, length, device="cuda")
        v[:, length // 2:length // 2 + 300] += 40
    check(v, call(v, None, k), None, k, 1.0)
    b = v.bfloat16()
    check(b, call(b, None, k), None, k, 1.0)


@pytest.mark.parametrize("length", [5, 1000, 70000])
def test_masks_infinities_and_nan(length):
    inf, k = math.inf, min(5, length)
    v = torch.randn(8, length, device="cuda")
    v[0] = -inf                                     # nothing left
    v[1, 1:] = -inf                                 # one left
    v[2, torch.rand(length, device="cuda") < 0.9] = -inf
    v[3, length // 2] = inf
    v[4, length - 1] = float("nan")
    v[5, 0], v[5, length - 1] = float("nan"), inf
    v[6] = -3.4e38                                  # the lowest finite value is not a mask
    v[7, ::2] = -3.4e38
    labels = torch.tensor([[0, length - 1, -1, length, 2 ** 31 - 1, -2 ** 31]] * 8, dtype=torch.int32, device="cuda")
    got = call(v, labels, k)
    check(v, got, labels, k, 1.0)
    assert float(got[1][0]) == 0.0 and bool((got[2][0] == -inf).all()) and got[3][0].tolist() == list(range(k))
    assert float(got[0][1, 0]) == 0.0 and float(got[1][1]) == 0.0


@pytest.mark.parametrize("kind", ["equal", "two values", "ascending", "descending", "crowded", "masked"])
@pytest.mark.parametrize("n,length", [(160, 5000), (150, 33000), (150, 131072)])
def test_hard_orders_in_rows_of_one_cta(kind, n, length):
    """more than two rows per SM are not split; crowded: thousands of the largest values in the shares of eight of 256 threads"""
    k = 32
    v = torch.randn(n, length, device="cuda")
    i = torch.arange(length, device="cuda")
    rows = slice(3, 9)
    if kind == "equal":
        v[rows] = 0.25
    elif kind == "two values":
        v[rows] = torch.randint(0, 2, (6, length), device="cuda").float()
    elif kind == "ascending":
        v[rows] = i.float() / 16
    elif kind == "descending":
        v[rows] = -i.float() / 16
    elif kind == "crowded":
        v[rows] += 50.0 * ((i // 4) % 256 < 8)
    else:
        v[rows, : length - 40] = -math.inf
    got = call(v, None, k)
    check(v[rows], [t[rows] for t in got], None, k, 1.0)
    b = v[:9].repeat(n // 9, 1).half()
    check(b[:9], [t[:9] for t in call(b, None, k)], None, k, 1.0)


def test_very_long_rows():
    v = torch.randn(2, 3000001, device="cuda") * 2
    labels = torch.tensor([[0], [3000000]], dtype=torch.int32, device="cuda")
    check(v, call(v, labels, 20), labels, 20, 1.0)


def test_large_logits_and_small_temperatures():
    v = torch.randn(4, 5000, device="cuda") * 1e4
    check(v, call(v, None, 5, 100.0), None, 5, 100.0)
    check(v, call(v, None, 5, 2.0 ** 120), None, 5, 2.0 ** 120)
    v = torch.randn(4, 5000, device="cuda") * 1e-3 + 1e3
    check(v, call(v, None, 5, 0.01), None, 5, 0.01)


def test_optional_outputs_and_launches():
    import deepracin_b200 as dr
    v = torch.randn(2, 300, device="cuda")
    lp, h, top, idx = call(v, None, 0, want_entropy=False)
    torch.cuda.synchronize()
    assert bool((h == 9.0).all())
    dr.lib.dRk_launch_count_reset()
    call(v, None, 3)
    assert dr.lib.dRk_launch_count() == 1


def test_same_answer_every_time():
    v = torch.randn(1, 131072, device="cuda")
    first = [t.clone() for t in call(v, None, 20)]
    for _ in range(10):
        for a, b in zip(first, call(v, None, 20)):
            assert torch.equal(a, b)


def test_streams_and_graph_capture():
    v, w = torch.randn(2, 40000, device="cuda"), torch.randn(700, 3000, device="cuda")
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    outs_v, outs_w = call(v, None, 8), call(w, None, 8)
    torch.cuda.synchronize()
    for _ in range(10):
        call(v, None, 8, stream=s1.cuda_stream, outs=outs_v)
        call(w, None, 8, stream=s2.cuda_stream, outs=outs_w)
    torch.cuda.synchronize()
    check(v, outs_v, None, 8, 1.0)
    check(w, outs_w, None, 8, 1.0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s1):
        call(v, None, 8, stream=s1.cuda_stream, outs=outs_v)
    for _ in range(3):
        v.copy_(torch.randn(2, 40000, device="cuda"))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        check(v, outs_v, None, 8, 1.0)


def test_long_rows_past_32_bits_of_bytes():
    """the last rows of a tensor of more than 4 GiB"""
    n, length = 9000, 131072
    if torch.cuda.mem_get_info()[0] < 8 << 30:
        pytest.skip("not enough memory")
    v = torch.zeros(n, length, dtype=torch.float32, device="cuda")
    v[-2:] = torch.randn(2, length, device="cuda")
    got = [t[-2:] for t in call(v, None, 4)]
    check(v[-2:], got, None, 4, 1.0)


# Rows of up to 8 or 16 vectors a lane are held by a warp: 32 partial sums of at most 16 + 8 + 7 additions, below the len / 128 + 64
# that check() allows.
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vectors", [8, 16])
def test_rows_around_what_a_warp_holds(vectors, dtype):
    most = 32 * vectors * (4 if dtype == torch.float32 else 8)
    g = torch.Generator().manual_seed(vectors)
    for length in (most - 9, most - 1, most, most + 1, most + 9):
        for n, shift in ((1, 0), (5, 1), (6, 3)):
            flat = torch.full((n * (length + shift) + shift,), math.nan, dtype=dtype, device="cuda")
            view = flat[shift:].view(n, length + shift)
            view[:, :length] = (torch.randn(n, length, generator=g) * 2.5).to(dtype).cuda()
            labels = torch.randint(-1, length + 1, (n, 40), generator=g, dtype=torch.int32).cuda()
            v = view[:, :length].contiguous()
            check(v, call(v, labels, 32, 1.25, ld=length + shift, ptr=view.data_ptr()), labels, 32, 1.25)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("length", [32, 289, 1024, 2048, 4096])
def test_hard_orders_in_rows_of_a_warp(length, dtype):
    g = torch.Generator().manual_seed(length)
    i = torch.arange(length)
    rows = [torch.full((length,), 1.5), torch.full((length,), -math.inf), torch.full((length,), math.nan), torch.full((length,), math.inf),
            torch.randint(0, 2, (length,), generator=g).float(), torch.where(torch.randint(0, 2, (length,), generator=g) == 1, 0.0, -0.0),
            i.float() / 64, -i.float() / 64, torch.where(i % 32 == 5, 8.0, 1.0) + torch.randn(length, generator=g),
            torch.where((i >= length // 2) & (i < length // 2 + 24), 9.0, 1.0), torch.where(i < 3, 1.0, -math.inf), torch.where(i == length - 1, math.nan, 0.0)]
    v = torch.stack(rows).to(dtype).cuda()
    for k in (1, 7, 32):
        labels = torch.randint(0, length, (len(rows), 2), generator=g, dtype=torch.int32).cuda()
        check(v, call(v, labels, k), labels, k, 1.0)


@pytest.mark.parametrize("kind", ["equal", "ascending", "crowded", "spread"])
@pytest.mark.parametrize("length", [5000, 33000, 131072])
def test_hard_orders_in_many_long_rows(length, kind):
    n, k = 600, 32
    if kind == "equal":
        v = torch.full((n, length), 1.5, device="cuda")
    elif kind == "ascending":
        v = (torch.arange(length, device="cuda").float() / 64).expand(n, length).contiguous()
    elif kind == "crowded":         # forty of the largest side by side in each row, elsewhere in each
        v = torch.randn(n, length, device="cuda")
        at = torch.randint(0, length - 40, (n, 1), device="cuda") + torch.arange(40, device="cuda")
        v.scatter_add_(1, at, torch.full(at.shape, 30.0, device="cuda"))
    else:
        v = torch.randn(n, length, device="cuda")
    got = [t[::97] for t in call(v, None, k)]
    check(v[::97], got, None, k, 1.0)
