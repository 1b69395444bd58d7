"""`rms_norm`: the residual's addition and the RMS norm in bf16, e4m3 and NVFP4, against the formula in 64 bits.

Bounds.  fp32 part: a sum of squares takes at most 64 additions in a thread, 10 over threads, and mean, root, reciprocal and two products
one rounding each, so v is within e = 2^-17 (128 roundings of 2^-24) of the exact one, relatively.  On top of that each format's own
rounding: half a step, 2^-8 of the value for bf16, 2^-4 for e4m3 (2^-10 of its unit among its subnormals), and for e2m1 a quarter below 2,
a half below 4, one below 6, in units of the block's scale (which is within half a step of e4m3 of maximum / 6, so a block's
largest value may pass 6 by 2^-4 of it, less than one)."""
import ctypes
import math
import sys

import pytest
import torch

from oracle import emulation as emu
from tests.helpers import gaussian

E = 2.0 ** -17
gpu = pytest.mark.gpu


def formula(x, weight, residual, eps):
    s = x.double() if residual is None else x.double() + residual.double()
    v = s / (s.square().mean(1, keepdim=True) + eps).sqrt()
    return s, v if weight is None else v * weight.double()


def inputs(m, k, residual=torch.bfloat16, weight=torch.bfloat16, seed=0):
    x = gaussian((m, k), seed, outlier_frac=0.005, outlier_mul=30).cuda()
    r = None if residual is None else gaussian((m, k), seed + 1, std=3).cuda().to(residual)
    if residual == torch.float32:
        r = r + gaussian((m, k), seed + 3, std=1e-3).cuda().float()
    w = None if weight is None else (1 + 0.3 * gaussian((k,), seed + 2).float()).cuda().to(weight)
    return x, w, r


def near_bf16(out, want, own=2.0 ** -8):
    got, want = out.double(), want.double()
    assert bool(((got - want).abs() <= want.abs() * (own * (1 + E) + E) + 2.0 ** -133).all())


def near_fp8(q, sf, v):
    m, k = v.shape
    assert q.shape == (m, -(-k // 16) * 16) and sf.shape == (-(-m // 16) * 16,)
    assert not q[:, k:].view(torch.uint8).any() and not sf[m:].any()
    want = v.abs().amax(1) / 448
    assert bool(((sf[:m].double() - want).abs() <= want * 2 * E).all())
    unit = sf[:m].double()[:, None]
    assert bool(((q[:, :k].double() * unit - v).abs() <= v.abs() * (2.0 ** -4 * (1 + 4 * E) + 4 * E) + unit * 2.0 ** -10).all())
    assert bool((q[:, :k].double().abs().amax(1) == 448).logical_or(want == 0).all())


def near_nvfp4(q, sf, g, v, layout):
    m, k = v.shape
    kp = -(-k // 64) * 64
    if layout == "128x4":
        pad = -(-m // 128) * 128
        assert sf.shape == (pad // 128, kp // 64, 32, 4, 4)
        scales = sf.double().permute(0, 3, 2, 1, 4).reshape(pad, kp // 16)      # tile [block][k64][row % 32][row / 32][4]
    else:
        pad = -(-m // 16) * 16
        assert sf.shape == (kp // 64, pad, 4)
        scales = sf.double().permute(1, 0, 2).reshape(pad, kp // 16)
    assert not scales[m:].any()
    full = torch.zeros(m, kp, dtype=torch.float64, device=v.device)
    full[:, :k] = v
    blocks = full.reshape(m, kp // 16, 16)
    want = blocks.abs().amax(2) / 6 / float(g)
    scales = scales[:m]
    assert bool(((scales - want.clamp(max=448)).abs() <= want.clamp(max=448) * (2.0 ** -4 + 4 * E) + 2.0 ** -10).all())
    unit = (scales * float(g))[:, :, None]
    codes = emu.e2m1_codes_to_float(emu.unpack_fp4(q)).double().reshape(m, kp // 16, 16)
    y = blocks.abs() / unit.clamp(min=1e-300)
    step = torch.where(y < 2, 0.25, torch.where(y < 4, 0.5, 1.0))
    inside = (want <= 448)[:, :, None] & (unit > 0)
    assert bool((((codes * unit - blocks).abs() <= (step + 16 * E * y + 16 * E) * unit) | ~inside).all())
    # a block whose scale is beyond e4m3 saturates, one whose scale rounds to nothing is zero
    top = (want > 464)[:, :, None] & (y > 6)
    assert bool((codes.abs() == 6)[top].all()) and not bool(codes[(unit == 0).expand_as(codes)].any())
    assert not codes.reshape(m, kp)[:, k:].any()


SHAPES = [(1, 8192), (1, 64), (3, 8), (5, 1), (2, 7), (17, 100), (33, 129), (130, 512), (129, 520), (9, 1024), (9, 1032), (70, 2048),
          (11, 4096), (7, 5120), (5, 8200), (3, 16384), (3, 16392), (2, 32768), (4, 5003), (2, 32761),
          (6, 511), (7, 514), (6, 1001), (3, 1027), (5, 2047), (5, 4095), (3, 8191), (2, 11003)]


@gpu
@pytest.mark.parametrize("m,k", SHAPES)
@pytest.mark.parametrize("residual,weight", [(torch.bfloat16, torch.bfloat16), (None, torch.float32), (torch.float32, None)])
def test_against_the_formula(m, k, residual, weight):
    from ac4k_kernel_b200 import ops
    x, w, r = inputs(m, k, residual, weight, seed=m + k)
    s, v = formula(x, w, r, 1e-6)
    got = ops.rms_norm(x, w, 1e-6, residual=r)
    out, total = got if r is not None else (got, None)
    near_bf16(out, v)
    if r is not None:
        assert total.dtype == r.dtype
        assert torch.equal(total, (x.float() + r.float()).to(r.dtype))

    got = ops.rms_norm(x, w, 1e-6, residual=r, precision="fp8e4m3", keep=True)
    assert torch.equal(got[2], out) and (r is None or torch.equal(got[3], total))
    near_fp8(got[0], got[1], v)

    g = (v.abs().max() / 2688).float()
    for layout in ("ac4k", "128x4"):
        got = ops.rms_norm(x, w, 1e-6, residual=r, precision="nvfp4", global_scale=g, keep=True, sf_layout=layout)
        assert got[2] is g and torch.equal(got[3], out) and (r is None or torch.equal(got[4], total))
        near_nvfp4(got[0], got[1], g, v, layout)
    small = g / 40                  # a scale that was calibrated too low: blocks saturate
    got = ops.rms_norm(x, w, 1e-6, residual=r, precision="nvfp4", global_scale=small)
    near_nvfp4(got[0], got[1], small, v, "ac4k")


@gpu
@pytest.mark.parametrize("k", [2048, 2056, 3000, 4096, 4104, 5120, 5128, 6144, 6152, 8192, 8200, 12288, 12296, 16384, 16392, 20000])
@pytest.mark.parametrize("residual,weight", [(torch.bfloat16, torch.bfloat16), (None, None), (torch.float32, torch.float32)])
def test_many_rows(k, residual, weight):
    """As many rows as take fewer threads each"""
    from ac4k_kernel_b200 import ops
    x, w, r = inputs(1030, k, residual, weight, seed=k)
    s, v = formula(x, w, r, 1e-6)
    got = ops.rms_norm(x, w, 1e-6, residual=r)
    out, total = got if r is not None else (got, None)
    near_bf16(out, v)
    assert r is None or torch.equal(total, (x.float() + r.float()).to(r.dtype))
    got = ops.rms_norm(x, w, 1e-6, residual=r, precision="fp8e4m3", keep=True)
    assert torch.equal(got[2], out) and (r is None or torch.equal(got[3], total))
    near_fp8(got[0], got[1], v)
    g = (v.abs().max() / 2688).float()
    got = ops.rms_norm(x, w, 1e-6, residual=r, precision="nvfp4", global_scale=g, sf_layout="128x4")
    near_nvfp4(got[0], got[1], g, v, "128x4")


@gpu
@pytest.mark.parametrize("k", [16384, 16381])
def test_rows_past_32_bits(k):
    """The last rows of every tensor begin behind 2^32 bytes"""
    from ac4k_kernel_b200 import ops
    m = 270000
    x = torch.randn((m, k), dtype=torch.bfloat16, device="cuda")
    _, w, _ = inputs(1, k, seed=2)
    out, sf, total = ops.rms_norm(x, w, 1e-6, residual=x, precision="fp8e4m3")
    for lo in (0, m - 100):
        s, v = formula(x[lo:lo + 100], w, x[lo:lo + 100], 1e-6)
        assert torch.equal(total[lo:lo + 100], (x[lo:lo + 100].float() * 2).bfloat16())
        near_fp8(out[lo:lo + 100], torch.cat([sf[lo:lo + 100], torch.zeros(12, device="cuda")]), v)


@gpu
@pytest.mark.parametrize("k", [64, 100, 1024, 2048, 4096, 8192, 16384, 32768])
@pytest.mark.parametrize("precision", [None, "fp8e4m3", "nvfp4"])
def test_a_row_is_the_same_alone_and_in_a_batch(k, precision):
    from ac4k_kernel_b200 import ops
    x, w, r = inputs(37, k, seed=k)
    g = torch.tensor(0.02, device="cuda") if precision == "nvfp4" else None
    many = ops.rms_norm(x, w, residual=r, precision=precision, global_scale=g)
    one = ops.rms_norm(x[20:21], w, residual=r[20:21], precision=precision, global_scale=g)
    assert torch.equal(many[0][20:21].view(torch.uint8), one[0].view(torch.uint8)) and torch.equal(many[-1][20:21], one[-1])
    if precision == "fp8e4m3":
        assert torch.equal(many[1][20], one[1][0])
    if precision == "nvfp4":
        assert torch.equal(many[1][:, 20].view(torch.uint8), one[1][:, 0].view(torch.uint8))


@gpu
@pytest.mark.parametrize("cut", [0, 1, 8])
@pytest.mark.parametrize("k", [512, 511])
def test_strided_rows(cut, k):
    """Rows that are a part of longer ones, at offsets that are and are not 16-byte aligned"""
    from ac4k_kernel_b200 import ops
    x, w, r = inputs(19, 700, seed=3)
    xs, rs, ws = x[:, cut:cut + k], r[:, cut:cut + k], w[cut:cut + k]
    s, v = formula(xs, ws, rs, 1e-5)
    out, total = ops.rms_norm(xs, ws.clone(), 1e-5, residual=rs)
    near_bf16(out, v)
    assert torch.equal(total, xs + rs)
    q, sf, _ = ops.rms_norm(xs, ws, 1e-5, residual=rs, precision="fp8e4m3")
    near_fp8(q, sf, v)
    rows = ops.rms_norm(x[::3, :k], None, 1e-5)
    near_bf16(rows, formula(x[::3, :k], None, None, 1e-5)[1])


@gpu
@pytest.mark.parametrize("k", [64, 63, 8192])
def test_rows_of_zeros_infinities_and_nan(k):
    from ac4k_kernel_b200 import ops
    x, w, _ = inputs(8, k, seed=1)
    x[1] = 0
    x[2] = 1e-38                       # (vanishes beside eps; the largest value is far above 2^-117)
    x[3, 5] = float("inf")
    x[4, 5] = float("nan")
    x[6] = 2.0 ** -130                 # subnormal: v is below 2^-117
    v = (x.float() * torch.rsqrt(x.float().square().mean(1, keepdim=True) + 1e-6) * w.float())
    out = ops.rms_norm(x, w)
    assert torch.equal(out.isnan(), v.isnan()) and not out[1].any()
    q, sf = ops.rms_norm(x, w, precision="fp8e4m3")
    assert not (q[1].view(torch.uint8) & 0x7F).any() and sf[1] == 0 and not (q[6].view(torch.uint8) & 0x7F).any() and sf[6] == 0
    for row in (3, 4):
        assert sf[row].isnan() and bool(q[row, :k].float().isnan().all())
    good = [0, 1, 2, 5, 7]
    _, v64 = formula(x[good], w, None, 1e-6)
    near_fp8(q[good], torch.cat([sf[good], sf[8:16], sf[8:11]]), v64)
    g = torch.tensor(1.0 / 64, device="cuda")
    p, psf, _ = ops.rms_norm(x, w, precision="nvfp4", global_scale=g)
    assert not psf[:, 1].view(torch.uint8).any() and not (p[1] & 0x77).any()
    for row in good:
        one, one_sf, _ = ops.rms_norm(x[row:row + 1], w, precision="nvfp4", global_scale=g)
        assert torch.equal(one[0], p[row]) and torch.equal(one_sf[:, 0].view(torch.uint8), psf[:, row].view(torch.uint8))
    zero = ops.rms_norm(x[good], w, precision="nvfp4", global_scale=torch.zeros((), device="cuda"))
    assert not (zero[0] & 0x77).any() and not zero[1].view(torch.uint8).any()
    inf_w = w.clone()
    inf_w[7] = float("inf")
    q, sf = ops.rms_norm(x[:1], inf_w, precision="fp8e4m3")
    assert not sf[0].isfinite() and bool(q[0, 7].float().isnan())

@gpu
@pytest.mark.parametrize("k", [8, 24, 40, 72, 5128, 7, 61, 65, 1001, 5121])
@pytest.mark.parametrize("rows", [6, 1030])
def test_padding_is_zeros_beside_nan_and_infinities(k, rows):
    """Rows whose scale is NaN or infinite: codes behind the last column are zeros all the same"""
    from ac4k_kernel_b200 import ops
    x, w, _ = inputs(rows, k, seed=k)
    x[0, k - 1] = float("nan")
    x[1, k // 2] = float("inf")
    x[2, k - 1] = -float("inf")
    x[3] = 0                           # with eps = 0 the formula's 0 / 0
    for eps in (1e-6, 0.0):
        q, sf = ops.rms_norm(x, w, eps, precision="fp8e4m3")
        assert not q[:, k:].view(torch.uint8).any() and not sf[rows:].any()
        assert bool(sf[:3].isnan().all()) and bool(sf[4:rows].isfinite().all()) and bool(sf[3] == 0 if eps else sf[3].isnan())
        for layout in ("ac4k", "128x4"):
            p, _, _ = ops.rms_norm(x, w, eps, precision="nvfp4", global_scale=torch.tensor(1.0 / 64, device="cuda"), sf_layout=layout)
            codes = torch.stack((p & 15, p >> 4), -1).reshape(rows, -1)
            assert not codes[:, k:].any()


@gpu
def test_no_rows():
    from ac4k_kernel_b200 import ops
    x = torch.empty((0, 128), dtype=torch.bfloat16, device="cuda")
    assert ops.rms_norm(x).shape == (0, 128)
    q, sf, total = ops.rms_norm(x, residual=x, precision="fp8e4m3")
    assert q.shape == (0, 128) and sf.shape == (0,) and total.shape == (0, 128)


@gpu
def test_in_place_residual_of_the_c_interface():
    """residual_out may be the residual itself, or x"""
    from ac4k_kernel_b200 import _cuda_ops
    for k in (4096, 999):
        x, w, r = inputs(21, k, seed=2)
        want, total = torch.empty_like(x), torch.empty_like(r)
        _cuda_ops.rms_norm(want, None, None, total, x, w, r, 1e-6)
        for target in ("residual", "x"):
            x2, r2, out = x.clone(), r.clone(), torch.empty_like(x)
            onto = r2 if target == "residual" else x2
            _cuda_ops.rms_norm(out, None, None, onto, x2, w, r2, 1e-6)
            assert torch.equal(out, want) and torch.equal(onto, total)


@gpu
def test_another_stream_and_a_graph():
    from ac4k_kernel_b200 import ops
    x, w, r = inputs(300, 2048, seed=4)
    want = ops.rms_norm(x, w, residual=r, precision="fp8e4m3")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = x * 2
        got = ops.rms_norm(y / 2, w, residual=r, precision="fp8e4m3")
    side.synchronize()
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.rms_norm(x, w, residual=r, precision="fp8e4m3")
    x.copy_(x.flip(0))
    r.copy_(r.flip(0))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got[0].view(torch.uint8), want[0].flip(0).view(torch.uint8)) and torch.equal(got[2], want[2].flip(0))


@gpu
def test_feeds_the_linear_layer():
    """norm -> linear in NVFP4 against the product of the values that the codes stand for"""
    from ac4k_kernel_b200 import ops
    x, w, r = inputs(50, 1024, seed=9)
    b = gaussian((512, 1024), 5, std=0.02).cuda()
    b4, b_sf, b_g = ops.quantize(b, 0, 1)
    g = torch.tensor(30.0 / 2688, device="cuda")
    q, sf, gs, _ = ops.rms_norm(x, w, residual=r, precision="nvfp4", global_scale=g)
    out = ops.linear(q, sf, gs, b4, b_sf, b_g)
    want = emu.linear_nvfp4_ref(q, sf, gs, b4, b_sf, b_g, out_dtype=torch.float64, accum_dtype=torch.float64)
    assert float((out.double() - want).norm() / want.norm()) < 2e-3


@gpu
def test_native_host_side_and_wrapper_agree(monkeypatch):
    from ac4k_kernel_b200 import ops
    from ac4k_kernel_b200.native import host_calls
    if host_calls is None:
        pytest.skip("the native host side is not built")
    module = sys.modules["ac4k_kernel_b200.ops.norm"]
    x, w, r = inputs(20, 320, seed=8)
    g = torch.tensor(0.01, device="cuda")
    calls = [dict(), dict(residual=r), dict(residual=r.float()), dict(precision="fp8e4m3"), dict(precision="fp8e4m3", keep=True, residual=r),
             dict(precision="nvfp4", global_scale=g), dict(precision="nvfp4", global_scale=g, sf_layout="128x4", keep=True, residual=r),
             dict(eps=1), dict(weight=None), dict(weight=w.float())]
    wrong = [dict(precision="int8"), dict(precision="nvfp4"), dict(global_scale=g), dict(keep=True), dict(residual=r[:5]), dict(residual=r.half()),
             dict(sf_layout="x"), dict(weight=w[:7]), dict(eps=-1.0), dict(x=x.half()), dict(x=x.t()), dict(x=x[0]), dict(x=x.cpu()),
             dict(weight=w.cpu()), dict(precision="nvfp4", global_scale=g.reshape(1)), dict(x=x[:, :0], weight=None)]
    for number, kw in enumerate(calls + wrong):
        res = []
        for path in (host_calls, None):
            monkeypatch.setattr(module, "host_calls", path)
            try:
                made = ops.rms_norm(kw.get("x", x), kw.get("weight", w), **{k: v for k, v in kw.items() if k not in ("x", "weight")})
                res.append([t.clone() for t in (made if isinstance(made, tuple) else (made,))])
            except Exception as e:
                res.append(type(e))
        if number >= len(calls):
            assert res[0] is res[1] and issubclass(res[0], Exception), (kw, res)
        else:
            assert len(res[0]) == len(res[1]) and all(torch.equal(a.reshape(-1).view(torch.uint8), b.reshape(-1).view(torch.uint8)) for a, b in zip(*res)), kw


def test_refusals_of_the_c_interface():
    """Bad arguments give negative codes before anything touches a device"""
    from ac4k_kernel_b200._lib import LIB, last_error
    P = 4096

    def call(out=P, sf=P, gs=P, precision=2, layout=0, normed=None, residual_out=P, x=P, residual=P, rdt=0, weight=P, wdt=0, eps=1e-6, m=4, k=64,
             xs=64, rs=64):
        return LIB.ac4k_rms_norm(out, sf, gs, precision, layout, normed, residual_out, x, residual, rdt, weight, wdt, eps, m, k, xs, rs, None)

    for kw, code in ((dict(precision=3), -4), (dict(layout=2), -4), (dict(rdt=1), -4), (dict(wdt=1), -4), (dict(m=-1), -2), (dict(k=0), -2),
                     (dict(xs=-64), -2), (dict(k=32769), -5), (dict(eps=-1.0), -2), (dict(eps=math.nan), -2), (dict(out=None), -1), (dict(x=None), -1),
                     (dict(sf=None), -1), (dict(gs=None), -1), (dict(residual=None), -1), (dict(precision=0, normed=P), -5), (dict(x=P + 1), -3),
                     (dict(residual=P + 2, rdt=2), -3), (dict(weight=P + 1), -3), (dict(sf=P + 2), -3), (dict(m=1 << 40), -2),
                     (dict(out=P + 2), -3), (dict(out=P + 2, precision=1), -3), (dict(out=P + 1, precision=0), -3)):
        assert call(**kw) == code, kw
        assert last_error()
    assert call(m=0, out=None) == 0
    assert isinstance(LIB.ac4k_rms_norm, ctypes._CFuncPtr)


def test_residual_out_that_overlaps_is_refused():
    """residual_out is the residual or x itself, in the same places and of the same type, or overlaps neither (no GPU: the refusal comes first)"""
    from ac4k_kernel_b200._lib import LIB, last_error
    Q = 1 << 20

    def call(residual_out, x=Q, residual=4 * Q, rdt=0, m=4, k=64, xs=64, rs=64):
        return LIB.ac4k_rms_norm(8 * Q, 9 * Q, 10 * Q, 2, 0, None, residual_out, x, residual, rdt, None, 0, 1e-6, m, k, xs, rs, None)

    for kw in (dict(residual_out=Q, xs=128), dict(residual_out=Q, rdt=2), dict(residual_out=Q + 128), dict(residual_out=Q - 128), dict(residual_out=4 * Q, rs=65),
               dict(residual_out=4 * Q, rs=0), dict(residual_out=4 * Q + 16), dict(residual_out=4 * Q + 256, rdt=2), dict(residual_out=Q, rdt=2, m=1)):
        assert call(**kw) == -2 and "residual_out" in last_error(), kw
    if not torch.cuda.is_available():          # past the checks: there is no device to launch on
        for kw in (dict(residual_out=Q), dict(residual_out=4 * Q), dict(residual_out=4 * Q, rdt=2), dict(residual_out=Q, xs=999, m=1), dict(residual_out=4 * Q, rs=7, m=1),
                   dict(residual_out=Q + 512, xs=64), dict(residual_out=2 * Q)):
            assert call(**kw) > 0, kw
