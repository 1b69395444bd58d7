"""`linear_grouped`: NVFP4 products with a weight per group of rows, against the products of the values that the codes stand for in 64 bits.

Bounds.  A product of two codes and their scales is exact in fp32; the sum over K takes one MMA of 64 products after another into an fp32
accumulator, each within 2^-22 of the terms so far, so 2^-16 of the sum of magnitudes for the K <= 4096 of these tests (2^-14 for the one of 16384, held to the same); alpha and bias round twice
more (2^-23); then one rounding to out: half a step, 2^-8 of the value for bf16, 2^-11 (2^-25 among its subnormals) for fp16, 2^-24 for fp32."""
import sys

import pytest
import torch

from oracle import emulation as emu
from tests.helpers import gaussian

gpu = pytest.mark.gpu
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def values(q, sf):
    """[.., rows, K] of packed codes and scales in the row layout, in float64"""
    rows = q.shape[-2]
    scales = sf.double().transpose(-3, -2)[..., :rows, :, :].flatten(-2)
    return emu.e2m1_codes_to_float(emu.unpack_fp4(q)).double() * scales.repeat_interleave(16, -1)


def case(lengths, n, k, lead=0, behind=0, seed=0, own_scales=False):
    from ac4k_kernel_b200 import ops
    e, t = len(lengths), lead + sum(lengths) + behind
    x = ops.quantize(gaussian((t, k), seed, outlier_frac=0.01, outlier_mul=20).cuda(), 0, 1)
    w = gaussian((e, n, k), seed + 1, std=0.05).cuda()
    if own_scales:
        each = [ops.quantize(w[i] * (i + 1), 0, 1) for i in range(e)]
        w = tuple(torch.stack(parts) for parts in zip(*each))
    else:
        w = ops.quantize(w, 1, 2)
    offsets = torch.tensor([lead] + [lead + sum(lengths[:i + 1]) for i in range(e)], dtype=torch.int32).cuda()
    return (*x, *w, offsets)


def check(out, x, x_sf, x_g, w, w_sf, w_g, offsets, bias=None):
    from ac4k_kernel_b200 import _lib
    assert _lib.device_status() == 0
    a, lo = values(x, x_sf), offsets.tolist()
    for e in range(w.shape[0]):
        rows = slice(lo[e], lo[e + 1])
        if lo[e + 1] <= lo[e]:
            continue
        b, g = values(w[e], w_sf[e]), float(x_g) * float(w_g if w_g.dim() == 0 else w_g[e])
        want, slack = a[rows] @ b.t() * g, a[rows].abs() @ b.abs().t() * g * 2.0 ** -16
        if bias is not None:
            want, slack = want + bias[e].double(), slack + bias[e].double().abs() * 2.0 ** -23
        slack = slack + want.abs() * 2.0 ** -22
        bound = slack + (want.abs() + slack) * HALF[out.dtype] + 2.0 ** -25
        assert bool(((out[rows].double() - want).abs() <= bound).all()), e


LENGTHS = [[1], [0, 1, 0, 0], [3, 0, 17, 1, 0, 40], [16, 16], [5, 33, 31], [64, 63, 1], [200, 0, 1, 65], [129, 127, 300], [0, 0, 1000, 3],
           [1, 2, 3, 4, 5, 6, 7, 8, 9]]


@gpu
@pytest.mark.parametrize("lengths", LENGTHS, ids=str)
@pytest.mark.parametrize("n,k", [(128, 64), (200, 320), (1024, 1024), (72, 4096), (8, 128), (129, 192)])
def test_against_the_formula(lengths, n, k):
    from ac4k_kernel_b200 import ops
    c = case(lengths, n, k, seed=n)
    check(ops.linear_grouped(*c), *c)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("bias_dtype", [None, torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("lengths", [[1, 2], [3, 20, 0, 31], [70, 5], [300, 200, 1]], ids=str)
def test_types_bias_and_scales(dtype, bias_dtype, lengths):
    from ac4k_kernel_b200 import ops
    c = case(lengths, 264, 1024, seed=5, own_scales=True)
    bias = None if bias_dtype is None else gaussian((len(lengths), 264), 9).cuda().to(bias_dtype)
    out = torch.empty((sum(lengths), 264), dtype=dtype, device="cuda")
    assert ops.linear_grouped(*c, bias=bias, out=out) is out
    check(out, *c, bias=bias)


@gpu
@pytest.mark.parametrize("lengths", [[1, 1, 1], [5, 0, 3], [17, 40], [100, 150], [700, 0, 300]], ids=str)
@pytest.mark.parametrize("lead,behind", [(0, 0), (1, 0), (0, 3), (2, 77), (130, 129)])
def test_rows_of_no_group(lengths, lead, behind):
    """Zeros in a new output, left as they are in a given one"""
    from ac4k_kernel_b200 import ops
    c = case(lengths, 136, 256, lead, behind, seed=7)
    rest = torch.ones(c[0].shape[0], dtype=torch.bool, device="cuda")
    rest[lead:lead + sum(lengths)] = False
    garbage = torch.full((c[0].shape[0], 136), float("nan"), dtype=torch.bfloat16, device="cuda")
    del garbage                     # (what a new output may be made of)
    out = ops.linear_grouped(*c)
    check(out, *c)
    assert not out[rest].any()
    given = torch.full_like(out, 7)
    ops.linear_grouped(*c, out=given)
    assert bool((given[rest] == 7).all()) and torch.equal(given[~rest], out[~rest])


@gpu
@pytest.mark.parametrize("m,n,k", [(1, 512, 1024), (16, 384, 512), (40, 512, 4096), (100, 256, 512), (300, 512, 1024), (1000, 1024, 2048)])
def test_one_group_is_the_linear_layer(m, n, k):
    from ac4k_kernel_b200 import ops
    c = case([m], n, k, seed=11)
    x, x_sf, x_g, w, w_sf, w_g, offsets = c
    out = ops.linear_grouped(*c)
    want = ops.linear(x, x_sf, x_g, w[0], w_sf[0], w_g)
    check(out, *c)
    assert float((out.double() - want.double()).norm() / want.double().norm()) < 2e-3


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lengths", [[100, 100, 0, 100], [129, 201, 63, 127], [125, 3, 128, 259], [385, 380, 1, 0], [53] * 40, [256, 256, 257, 511]], ids=str)
@pytest.mark.parametrize("n,k", [(520, 576), (136, 4096)])
def test_groups_that_fill_half_a_tile(lengths, n, k, dtype):
    """A pair's second half has rows of the group, a few of them or none, whatever row the group begins at"""
    from ac4k_kernel_b200 import ops
    c = case(lengths, n, k, lead=1, behind=2, seed=n + len(lengths))
    out = torch.full((c[0].shape[0], n), 7.0, dtype=dtype, device="cuda")
    check(ops.linear_grouped(*c, out=out), *c)
    assert bool((out[:1] == 7).all()) and bool((out[-2:] == 7).all())

@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lengths", [[100, 100, 0, 100], [129, 201, 63, 127], [125, 3, 128, 259], [385, 380, 1, 0], [53] * 40, [256, 256, 257, 511]], ids=str)
@pytest.mark.parametrize("n,k", [(136, 576), (264, 960)])
def test_groups_that_fill_half_a_tile_uncut(lengths, n, k, dtype):
    """As above with a K that is not cut into slices (fewer than eight stages of 256), so that all of them are tiles of CTA pairs"""
    from ac4k_kernel_b200 import ops
    c = case(lengths, n, k, lead=1, behind=2, seed=n + len(lengths))
    out = torch.full((c[0].shape[0], n), 7.0, dtype=dtype, device="cuda")
    check(ops.linear_grouped(*c, out=out), *c)
    assert bool((out[:1] == 7).all()) and bool((out[-2:] == 7).all())


@gpu
def test_a_group_is_the_same_alone_and_among_others():
    """Its rows' place, the other groups' contents (NaN scales among them) and empty groups change nothing"""
    from ac4k_kernel_b200 import ops
    lengths = [7, 0, 90, 33, 2]
    x, x_sf, x_g, w, w_sf, w_g, offsets = case(lengths, 256, 512, seed=13)
    out = ops.linear_grouped(x, x_sf, x_g, w, w_sf, w_g, offsets)
    sf, wsf = x_sf.clone(), w_sf.clone()
    sf.view(torch.uint8)[:, :7] = 0x7F
    sf.view(torch.uint8)[:, 97:132] = 0x7F
    for e in (0, 1, 3, 4):
        wsf.view(torch.uint8)[e] = 0x7F
    other = ops.linear_grouped(x, sf, x_g, w, wsf, w_g, offsets)
    assert torch.equal(other[7:97], out[7:97])
    assert bool(other[:7].isnan().all()) and bool(other[97:].isnan().all())


@gpu
@pytest.mark.parametrize("each", [1, 40])
def test_weights_past_32_bits(each):
    """5.4 GB of codes: the last groups' weights begin behind 2^32 bytes"""
    from ac4k_kernel_b200 import ops
    e, n, k = 40, 16384, 16384
    x = ops.quantize(gaussian((e * each, k), 41).cuda(), 0, 1)
    w = torch.randint(0, 256, (e, n, k // 2), dtype=torch.uint8, device="cuda")
    w_sf = torch.randint(0x28, 0x40, (e, k // 64, n, 4), dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    w_g = torch.tensor(0.01, device="cuda")
    offsets = torch.arange(0, e * each + 1, each, dtype=torch.int32, device="cuda")
    out = ops.linear_grouped(*x, w, w_sf, w_g, offsets)
    for g in (0, e - 2, e - 1):
        for n0 in (0, n - 256):
            part = torch.tensor([each * g, each * (g + 1)], dtype=torch.int32)
            check(out[:, n0:n0 + 256], *x, w[g:g + 1, n0:n0 + 256], w_sf[g:g + 1, :, n0:n0 + 256], w_g, part)


@gpu
def test_many_groups():
    from ac4k_kernel_b200 import ops
    g = torch.Generator().manual_seed(3)
    lengths = [int(v) if v > 0 else 0 for v in torch.randint(-8, 5, (700,), generator=g)]
    c = case(lengths, 64, 64, lead=2, behind=1, seed=17)
    check(ops.linear_grouped(*c), *c)

@gpu
@pytest.mark.parametrize("lead,behind", [(0, 0), (3, 5)])
@pytest.mark.parametrize("groups,longest", [(129, 60), (300, 40), (700, 30)])
def test_more_groups_than_ranges_of_the_table(groups, longest, lead, behind):
    """The CTA-pair kernel's table has 128 entries: several groups an entry, empty ones among them"""
    from ac4k_kernel_b200 import ops
    g = torch.Generator().manual_seed(groups)
    lengths = torch.randint(-longest // 8, longest + 1, (groups,), generator=g).clamp(min=0).tolist()
    assert sum(lengths) > 9 * groups             # (what sends them to the pairs at this K)
    c = case(lengths, 264, 256, lead, behind, seed=groups)
    out = torch.full((c[0].shape[0], 264), 7.0, dtype=torch.bfloat16, device="cuda")
    check(ops.linear_grouped(*c, out=out), *c)
    rest = torch.ones(out.shape[0], dtype=torch.bool, device="cuda")
    rest[lead:lead + sum(lengths)] = False
    assert bool((out[rest] == 7).all())
    assert not ops.linear_grouped(*c)[rest].any()

@gpu
@pytest.mark.parametrize("groups,each", [(200, 30), (3, 20000)])
def test_more_tiles_than_are_listed(groups, each):
    """More than 48 tiles of 256 x 256 for each of 74 pairs (3552): the rest are looked up as they come"""
    from ac4k_kernel_b200 import ops
    lengths = [each + i % 3 for i in range(groups)]
    c = case(lengths, 8192, 64, seed=each)
    assert groups * -(-each // 256) * 32 > 3552
    check(ops.linear_grouped(*c), *c)


@gpu
def test_nothing_to_do():
    from ac4k_kernel_b200 import ops
    x, x_sf, x_g, w, w_sf, w_g, offsets = case([3, 4], 128, 128, seed=19)
    zero = torch.zeros_like(offsets)
    assert not ops.linear_grouped(x, x_sf, x_g, w, w_sf, w_g, zero).any()
    given = torch.full((7, 128), 7.0, device="cuda")
    assert bool((ops.linear_grouped(x, x_sf, x_g, w, w_sf, w_g, zero, out=given) == 7).all())
    assert ops.linear_grouped(x[:0], x_sf[:, :0].contiguous(), x_g, w, w_sf, w_g, zero).shape == (0, 128)
    assert not ops.linear_grouped(x, x_sf, x_g, w[:0], w_sf[:0], w_g, zero[:1]).any()


@gpu
@pytest.mark.parametrize("t,behind", [(60, 60), (700, 60)])
def test_offsets_that_are_none(t, behind):
    """Offsets past the rows, negative and descending ones reach no memory of others"""
    from ac4k_kernel_b200 import ops
    x, x_sf, x_g, w, w_sf, w_g, _ = case([t // 3] * 3, 128, 256, seed=23)
    rows = x.shape[0]
    big = torch.full((rows + 2 * behind, 128), 7.0, dtype=torch.bfloat16, device="cuda")
    for bad in ([-5, 10, 20, rows], [0, 10, 20, 10 ** 6], [0, 20, 10, 30], [30, 20, 10, 0], [2 ** 31 - 1, -2 ** 31, 2 ** 31 - 1, 5], [0, rows, 0, rows]):
        offsets = torch.tensor(bad, dtype=torch.int32, device="cuda")
        ops.linear_grouped(x, x_sf, x_g, w, w_sf, w_g, offsets, out=big[behind:behind + rows])
        torch.cuda.synchronize()
        assert bool((big[:behind] == 7).all()) and bool((big[behind + rows:] == 7).all())

@gpu
@pytest.mark.parametrize("n", [136, 520])
@pytest.mark.parametrize("fill", [False, True])
def test_offsets_that_are_none_in_pairs(n, fill):
    """As above, at widths and lengths of the CTA-pair kernel, which has its own lookup; lists without any row among them"""
    from ac4k_kernel_b200 import _cuda_ops, _lib, ops
    x, x_sf, x_g, w, w_sf, w_g, right = case([250, 0, 200, 250], n, 256, seed=23)
    rows, behind = x.shape[0], 60
    big = torch.full((rows + 2 * behind, n), 7.0, dtype=torch.bfloat16, device="cuda")
    out = big[behind:behind + rows]
    if out.data_ptr() % 16:
        pytest.fail("the rows begin on 16 bytes")
    want = ops.linear_grouped(x, x_sf, x_g, w, w_sf, w_g, right)
    for bad in ([-5, 10, 20, 30, rows], [0, 10, 20, 10 ** 6, 10 ** 6], [0, 20, 10, 30, 30], [30, 20, 10, 0, 5], [2 ** 31 - 1, -2 ** 31, 2 ** 31 - 1, 5, 9],
                [0, rows, 0, rows, 0], [rows] * 5, [0] * 5, [300] * 5, [-7] * 5):
        out.fill_(5.0)
        offsets = torch.tensor(bad, dtype=torch.int32, device="cuda")
        _cuda_ops.linear_nvfp4_grouped(out, x, x_sf, x_g, w, w_sf, w_g, offsets, None, fill)
        assert _lib.device_status() == 0
        assert bool((big[:behind] == 7).all()) and bool((big[behind + rows:] == 7).all())
        if len(set(bad)) == 1:                          # no group has a row
            assert bool((out == (0.0 if fill else 5.0)).all())
    _cuda_ops.linear_nvfp4_grouped(out, x, x_sf, x_g, w, w_sf, w_g, right, None, fill)
    assert torch.equal(out, want)


@gpu
def test_same_result_each_time_streams_and_graphs():
    from ac4k_kernel_b200 import ops
    small, large = case([1, 0, 2, 1], 512, 2048, seed=29), case([300, 0, 700], 512, 512, seed=31)
    want, want_l = ops.linear_grouped(*small), ops.linear_grouped(*large)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(20):
        with torch.cuda.stream(side):
            other = ops.linear_grouped(*large)
        assert torch.equal(ops.linear_grouped(*small), want)
        side.synchronize()
        assert torch.equal(other, want_l)
    graphs = []
    for args in (small, large):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = ops.linear_grouped(*args)
        graphs.append((graph, out))
    for _ in range(5):
        for _, out in graphs:
            out.zero_()
        torch.cuda.synchronize()
        graphs[0][0].replay()
        with torch.cuda.stream(side):
            graphs[1][0].replay()
        torch.cuda.synchronize()
        assert torch.equal(graphs[0][1], want) and torch.equal(graphs[1][1], want_l)
    # other lengths in the same captured call
    x, x_sf, x_g, w, w_sf, w_g, offsets = large
    offsets.copy_(torch.tensor([0, 10, 900, 1000], dtype=torch.int32))
    graphs[1][0].replay()
    torch.cuda.synchronize()
    check(graphs[1][1], *large)


@gpu
def test_norm_experts_and_back():
    """norm to NVFP4 with the rows sorted by expert -> the experts' first product -> its output quantised -> their second"""
    from ac4k_kernel_b200 import ops
    g = torch.Generator().manual_seed(5)
    tokens, experts, k, inner = 90, 6, 256, 512
    x, r = gaussian((tokens, k), 1).cuda(), gaussian((tokens, k), 2).cuda()
    which = torch.randint(0, experts - 1, (tokens,), generator=g).cuda()
    order = which.argsort(stable=True)
    offsets = torch.cat([torch.zeros(1, device="cuda"), torch.bincount(which, minlength=experts).cumsum(0)]).int()
    up, down = (ops.quantize(gaussian(s, 3, std=0.05).cuda(), 1, 2) for s in ((experts, inner, k), (experts, k, inner)))
    q, sf, gs, total = ops.rms_norm(x[order], residual=r[order], precision="nvfp4", global_scale=torch.tensor(12 / 2688, device="cuda"))
    h = ops.linear_grouped(q, sf, gs, *up, offsets)
    check(h, q, sf, gs, *up, offsets)
    h4 = ops.quantize(h, 0, 1)
    out = ops.linear_grouped(*h4, *down, offsets)
    check(out, *h4, *down, offsets)
    back = torch.empty_like(out)
    back[order] = out
    assert torch.equal(total, x[order] + r[order]) and bool(back.isfinite().all())


@gpu
def test_native_host_side_and_wrapper_agree(monkeypatch):
    from ac4k_kernel_b200 import ops
    from ac4k_kernel_b200.native import host_calls
    if host_calls is None:
        pytest.skip("the native host side is not built")
    module = sys.modules["ac4k_kernel_b200.ops.linear"]
    names = ("x", "x_scale", "x_global_scale", "weight", "weight_scale", "weight_global_scale", "offsets")
    good = dict(zip(names, case([5, 20], 128, 192, seed=37)))
    bias = gaussian((2, 128), 1).cuda()
    new = lambda dt, m=25: torch.empty((m, 128), dtype=dt, device="cuda")  # noqa: E731
    calls = [dict(), dict(bias=bias), dict(bias=bias.float()), dict(out=new(torch.half)), dict(weight_global_scale=torch.ones(2, device="cuda"))]
    x, w = good["x"], good["weight"]
    wrong = [dict(x=x[:8]), dict(x=x.int()), dict(x=x[:, :64]), dict(x=x.cpu()), dict(weight=w[:1]), dict(weight=w[0]), dict(weight=w.cpu()),
             dict(x_scale=good["x_scale"][:, :16]), dict(weight_scale=good["weight_scale"][0]), dict(offsets=good["offsets"].long()),
             dict(offsets=good["offsets"][:2]), dict(offsets=good["offsets"].cpu()), dict(x_global_scale=torch.ones(1, device="cuda")),
             dict(weight_global_scale=torch.ones(3, device="cuda")), dict(bias=bias[:1]), dict(bias=bias[0]), dict(bias=bias.double()),
             dict(out=new(torch.double)), dict(out=new(torch.half, 24)), dict(out=new(torch.half, 50)[::2]), dict(bias=bias.cpu())]
    for number, kw in enumerate(calls + wrong):
        res = []
        for path in (host_calls, None):
            monkeypatch.setattr(module, "host_calls", path)
            try:
                res.append(ops.linear_grouped(**{**good, **kw}).clone())
            except Exception as e:
                res.append(type(e))
        if number >= len(calls):
            assert res[0] is res[1] and issubclass(res[0], Exception), (number, res)
        else:
            assert torch.equal(res[0], res[1]), number


def test_refusals_of_the_c_interface():
    """Bad arguments give negative codes before anything touches a device"""
    from ac4k_kernel_b200._lib import LIB, last_error
    P = 4096

    def call(d=P, dt=0, a=P, asf=P, ags=P, b=P, bsf=P, bgs=P, per=0, bias=None, bdt=0, offsets=P, fill=0, m=4, e=2, n=64, k=64):
        return LIB.ac4k_linear_nvfp4_grouped(d, dt, a, asf, ags, b, bsf, bgs, per, bias, bdt, offsets, fill, m, e, n, k, None)

    for kw, code in ((dict(dt=3), -4), (dict(bias=P, bdt=7), -4), (dict(m=-1), -2), (dict(e=-1), -2), (dict(k=0), -2), (dict(k=80), -2),
                     (dict(e=1 << 20, n=1 << 20), -2), (dict(d=None), -1), (dict(a=None), -1), (dict(bgs=None), -1), (dict(offsets=None), -1),
                     (dict(d=P + 4), -3), (dict(bsf=P + 8), -3), (dict(offsets=P + 2), -3), (dict(bias=P + 1), -3), (dict(bias=P + 2, bdt=2), -3)):
        assert call(**kw) == code, kw
        assert last_error()
    assert call(m=0) == 0 and call(n=0) == 0 and call(e=0, a=None) == 0
