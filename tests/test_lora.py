"""`lora`: the adapters of a batch of requests added to a projection's output, against the formula in 64 bits.

Bounds.  A x: fp32 sums of exact products, at most K / 16 additions of MMAs of 16 products (each MMA sums within 2^-21 of its largest
terms), so within 2^-15 of the sum of the magnitudes |A| |x| for the K of these tests.  A x split into two bf16 parts: 2^-16 of it.
B of that: the same again over R.  So the sum added to y is within 2^-13 of scaling * |B| (|A| |x|), and out rounds once: half a step, 2^-8
of the value for bf16, 2^-11 for fp16 (2^-25 among its subnormals), 2^-24 for fp32."""
import sys

import pytest
import torch

from tests.helpers import gaussian

gpu = pytest.mark.gpu
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def case(lengths, adapters, k, n, rank, count, dtype=torch.bfloat16, lead=0, behind=0, seed=0, scaling=True):
    t = lead + sum(lengths) + behind
    offsets = torch.tensor([lead] + [lead + sum(lengths[:i + 1]) for i in range(len(lengths))], dtype=torch.int32).cuda()
    x = gaussian((t, k), seed, outlier_frac=0.01, outlier_mul=20).cuda()
    y = gaussian((t, n), seed + 1).cuda().to(dtype)
    a = gaussian((count, rank, k), seed + 2, std=k ** -0.5).cuda()
    b = gaussian((count, n, rank), seed + 3, std=0.2).cuda()
    s = (0.5 + torch.arange(count, dtype=torch.float32) / max(1, count)).cuda() if scaling else None
    return y, x, a, b, offsets, torch.tensor(adapters, dtype=torch.int32).cuda(), s


def check(out, y, x, a, b, offsets, adapters, s):
    want, slack = y.double().clone(), torch.zeros_like(y, dtype=torch.float64)
    lo = offsets.tolist()
    for i, j in enumerate(adapters.tolist()):
        rows = slice(lo[i], lo[i + 1])
        if 0 <= j < a.shape[0] and lo[i + 1] > lo[i]:
            f = 1.0 if s is None else float(s[j])
            want[rows] += f * (x[rows].double() @ a[j].double().t()) @ b[j].double().t()
            slack[rows] = abs(f) * (x[rows].double().abs() @ a[j].double().abs().t()) @ b[j].double().abs().t()
    assert out.dtype == y.dtype and out.shape == y.shape
    bound = slack * 2.0 ** -13
    bound = bound + (want.abs() + bound) * HALF[y.dtype] + 2.0 ** -25
    assert bool(((out.double() - want).abs() <= bound).all())


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rank", [1, 4, 8, 12, 16, 24, 32, 64, 100, 128])
@pytest.mark.parametrize("lengths", [[1], [1, 1, 1, 1, 1], [3, 0, 17, 1, 0, 40], [200, 0, 1, 65], [64, 64]])
def test_against_the_formula(dtype, rank, lengths):
    from ac4k_kernel_b200 import ops
    c = case(lengths, [i % 3 for i in range(len(lengths))], 640, 328, rank, 3, dtype, seed=rank)
    check(ops.lora(*c), *c)

@gpu
@pytest.mark.parametrize("rank", [1, 16, 24, 64, 128])
@pytest.mark.parametrize("lengths", [[1], [1, 1, 5, 2], [100], [64, 130]], ids=str)
@pytest.mark.parametrize("k,n", [(512, 328), (500, 37)])
def test_fp32_rows_get_all_of_the_sum(k, n, lengths, rank):
    """Whole numbers: products up to 2^14, A x up to 2^23 (some 2^17), sums of B of them below 2^24 with entries of 0 and +-1 in B, eight of them
    a column at most.  Nothing is rounded on the way in fp32, so out is exact: what is lost of A x shows."""
    from ac4k_kernel_b200 import ops
    y, x, a, b, offsets, adapters, _ = case(lengths, [i % 2 for i in range(len(lengths))], k, n, rank, 2, torch.float32)
    g = torch.Generator().manual_seed(rank + k)
    x = torch.randint(-128, 129, x.shape, generator=g).bfloat16().cuda()
    a = torch.randint(-128, 129, a.shape, generator=g).bfloat16().cuda()
    b = torch.randint(-1, 2, b.shape, generator=g).bfloat16().cuda()
    b[:, :, 8:] = 0
    y = torch.randint(-1000, 1000, y.shape, generator=g).float().cuda()
    want, lo = y.double().clone(), offsets.tolist()
    for i, j in enumerate(adapters.tolist()):
        low = x[lo[i]:lo[i + 1]].double() @ a[j].double().t()
        assert float(low.abs().max()) * 8 < 2 ** 24 - 1000
        want[lo[i]:lo[i + 1]] += low @ b[j].double().t()
    assert torch.equal(ops.lora(y, x, a, b, offsets, adapters).double(), want)


@gpu
@pytest.mark.parametrize("k,n", [(8, 8), (1, 1), (33, 65), (40, 200), (1000, 36), (4096, 1024), (5000, 1416), (130, 2050)])
@pytest.mark.parametrize("rank", [3, 16, 64])
@pytest.mark.parametrize("lengths", [[2, 1, 1], [100, 37]])
def test_odd_sizes(k, n, rank, lengths):
    from ac4k_kernel_b200 import ops
    c = case(lengths, [1, 0, 1][:len(lengths)], k, n, rank, 2, seed=k + n)
    check(ops.lora(*c), *c)


@gpu
@pytest.mark.parametrize("rank", [16, 32, 64, 128])
@pytest.mark.parametrize("lengths", [[1], [40], [200], [1] * 9, [16, 2, 30, 5], [70, 500, 3, 130], [700] * 6], ids=lambda v: f"{len(v)}x{v[0]}")
def test_clusters_of_every_size(lengths, rank):
    """Few tiles take a cluster of 16 blocks each, more of them smaller ones down to a single block; slices that end inside K and N"""
    from ac4k_kernel_b200 import ops
    c = case(lengths, [i % 3 for i in range(len(lengths))], 4872, 4424, rank, 3, seed=rank + len(lengths))
    check(ops.lora(*c), *c)

@gpu
@pytest.mark.parametrize("rank", [16, 32, 64, 128])
@pytest.mark.parametrize("tiles", [56, 72, 95, 108, 140, 190, 220, 290, 400])
def test_clusters_of_few_blocks(tiles, rank):
    """A prompt of so many tiles of 64 rows that a cluster has 1 to 5 blocks, or more of them where four fit on an SM: 148 SMs hold 592 blocks of ranks 16 and
    32, 444 of rank 64 and 296 of rank 128"""
    from ac4k_kernel_b200 import ops
    lengths = [64 * tiles - 70, 0, 33]
    c = case(lengths, [0, 1, 1], 1304, 1288, rank, 2, lead=2, seed=tiles)
    check(ops.lora(*c), *c)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n,cut", [(2504, 0), (2504, 8), (2501, 0), (600, 4)])
@pytest.mark.parametrize("tokens", [2, 90])
def test_long_rows_without_an_adapter(dtype, n, cut, tokens):
    from ac4k_kernel_b200 import ops
    y, x, a, b, offsets, adapters, s = case([tokens] * 4, [-1, 0, -1, 1], 256, n, 16, 2, dtype, lead=3, behind=20, seed=15)
    c = (y[:, cut:], x, a, b[:, cut:].contiguous(), offsets, adapters, s)
    whole = torch.full((y.shape[0], n + 64), 7.0, dtype=dtype, device="cuda")
    out = ops.lora(*c, out=whole[:, 8:8 + n - cut])
    check(out, *c)
    without = torch.ones(y.shape[0], dtype=torch.bool, device="cuda")
    for i in (1, 3):
        without[3 + i * tokens:3 + (i + 1) * tokens] = False
    assert torch.equal(out[without], c[0][without])
    assert bool((whole[:, :8] == 7).all()) and bool((whole[:, 8 + n - cut:] == 7).all())


@gpu
@pytest.mark.parametrize("tokens", [1, 6, 100])
def test_rows_without_an_adapter_stay_as_they_are(tokens):
    """Requests without one, an index that there is no adapter of, rows in front of the first request and behind the last"""
    from ac4k_kernel_b200 import ops
    y, x, a, b, offsets, adapters, s = case([tokens, tokens, 0, tokens, tokens], [-1, 1, 0, 7, 0], 256, 200, 16, 2, lead=5, behind=70, seed=3)
    x[:5] = float("nan")
    x[-70:] = float("inf")
    x[5:5 + tokens] = float("nan")
    y[0, 0], y[-1, -1], y[5, 3] = float("nan"), float("inf"), float("nan")
    rows = torch.ones(y.shape[0], dtype=torch.bool, device="cuda")
    rows[5 + tokens:5 + 2 * tokens] = False
    rows[5 + 3 * tokens:5 + 4 * tokens] = False
    bits = y.view(torch.int16).clone()
    out = ops.lora(y, x, a, b, offsets, adapters, s)
    assert torch.equal(out.view(torch.int16)[rows], bits[rows])
    assert torch.equal(y.view(torch.int16), bits)
    own = ops.lora(y, x, a, b, offsets, adapters, s, out=y)
    assert own is y and torch.equal(y.view(torch.int16), out.view(torch.int16))


@gpu
def test_nan_stays_in_its_row_and_its_adapter():
    from ac4k_kernel_b200 import ops
    y, x, a, b, offsets, adapters, s = case([20, 20, 20], [0, 1, 2], 128, 64, 8, 3, seed=4)
    clean = ops.lora(y, x, a, b, offsets, adapters, s)
    a[1] = float("nan")
    x[3, 7] = float("nan")
    out = ops.lora(y, x, a, b, offsets, adapters, s)
    hit = torch.zeros(60, dtype=torch.bool, device="cuda")
    hit[20:40] = True
    hit[3] = True
    assert torch.equal(out[~hit], clean[~hit]) and bool(out[hit].isnan().all())
    x[3, 7] = float("inf")          # A x is infinite: what B makes of it is an infinity or a NaN, as in the formula
    a[0], b[0] = 1.0, 1.0
    assert bool((ops.lora(y, x, a, b, offsets, adapters, s)[3] == float("inf")).all())


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rank", [3, 16, 40, 128])
@pytest.mark.parametrize("exact", [True, False])
def test_infinite_weights_give_infinities(exact, rank, dtype):
    """An infinite B takes its sign from A x, whatever A x leaves behind where it is cut into parts of 8 bits: nothing (`exact`: A x are 7-bit
    numbers, some of them 0) or a rest of the one or the other sign.  NaN only where the formula has 0 * infinity or infinities of both signs."""
    from ac4k_kernel_b200 import ops
    y, x, a, b, offsets, adapters, _ = case([1, 7, 90], [0, 1, 0], 256, 136, rank, 2, dtype, seed=rank)
    if exact:
        x = (torch.arange(x.numel(), device="cuda").reshape(x.shape) * 37 % 129 - 64).bfloat16()
        a.zero_()
        for r in range(rank):
            a[:, r, (5 * r + 1) % 256] = 1.0
    for j in range(2):
        b[j, 3, 0] = float("inf")
        b[j, 4, 1] = -float("inf")
        b[j, 70, 0], b[j, 70, 2] = float("inf"), float("inf")
        b[j, 135, rank - 1] = float("inf")
    want, lo = y.double().clone(), offsets.tolist()
    for i, j in enumerate(adapters.tolist()):
        low = x[lo[i]:lo[i + 1]].double() @ a[j].double().t()
        want[lo[i]:lo[i + 1]] += (low[:, None, :] * b[j].double()).sum(-1)        # (no product that a library skips)
    out = ops.lora(y, x, a, b, offsets, adapters).double()
    assert torch.equal(out.isnan(), want.isnan())
    assert torch.equal(out == float("inf"), want == float("inf")) and torch.equal(out == -float("inf"), want == -float("inf"))
    assert bool(want.isinf().any()) and (not exact or bool(want.isnan().any()))


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("cut", [0, 1, 8])
def test_strides(dtype, cut):
    from ac4k_kernel_b200 import ops
    y, x, a, b, offsets, adapters, s = case([1, 50, 9], [1, 0, 1], 300, 260, 16, 2, dtype, seed=6)
    c = (y[:, cut:cut + 240], x[:, cut:cut + 200], a[:, :, :200].contiguous(), b[:, :240].contiguous(), offsets, adapters, s)
    check(ops.lora(*c), *c)
    big = torch.full((60, 512), 7.0, dtype=dtype, device="cuda")
    out = ops.lora(*c, out=big[:, 16:256])
    check(out, *c)
    assert bool((big[:, :16] == 7).all()) and bool((big[:, 256:] == 7).all())
    want = out.clone()
    assert torch.equal(ops.lora(*c, out=c[0]), want)
    wide = (y[:1, cut:cut + 240].expand(60, 240), *c[1:])           # one row of y for all
    check(ops.lora(*wide), *wide)

@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n", [48, 45])
def test_one_row_in_place_whatever_its_stride(n, dtype):
    """A single row's stride means nothing: out at y's address is y"""
    from ac4k_kernel_b200 import ops
    y, x, a, b, offsets, adapters, s = case([1], [1], 64, n, 8, 2, dtype, seed=21)
    want = ops.lora(y, x, a, b, offsets, adapters, s)
    big = torch.full((3, 200), 7.0, dtype=dtype, device="cuda")
    big[0, :n] = y[0]
    out = big[0, :n].unsqueeze(0)
    row = big[:1, :n].as_strided((1, n), (200, 1))
    assert row.data_ptr() == out.data_ptr()
    for given in (out.as_strided((1, n), (n, 1)), row, out.as_strided((1, n), (1, 1))):
        big[0, :n] = y[0]
        assert ops.lora(row, x, a, b, offsets, adapters, s, out=given) is given
        assert torch.equal(given, want) and bool((big[0, n:] == 7).all())
        assert torch.equal(ops.lora(row, x, a[:0], b[:0], offsets, adapters, out=given), want)
    far = torch.zeros((1, 64), dtype=torch.bfloat16, device="cuda").as_strided((1, 64), (1, 1))      # one row of x, whatever its stride
    far.copy_(x)
    assert torch.equal(ops.lora(y, far, a, b, offsets, adapters, s), want)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rank", [4, 16, 32, 64, 128])
@pytest.mark.parametrize("requests,count,longest", [(2, 1, 1), (9, 1, 1), (50, 3, 1), (129, 64, 2), (254, 5, 3), (255, 5, 3), (40, 2, 30), (64, 20, 1)])
def test_requests_that_share_adapters(requests, count, longest, rank, dtype):
    """Rows of one adapter from all over the batch, empty requests, requests without an adapter and rows of no request among them"""
    from ac4k_kernel_b200 import ops
    g = torch.Generator().manual_seed(requests + rank)
    lengths = torch.randint(0 if longest > 1 else 1, longest + 1, (requests,), generator=g).tolist()
    adapters = torch.randint(-1 if requests > 9 else 0, count + (requests > 50), (requests,), generator=g).tolist()
    y, x, a, b, offsets, which, s = case(lengths, adapters, 712, 392, rank, count, dtype, lead=5, behind=19, seed=requests)
    x[:5], x[-19:] = float("nan"), float("nan")
    c = (y[:, 8:], x[:, 8:], a[:, :, 8:].contiguous(), b[:, 8:].contiguous(), offsets, which, s)
    out = ops.lora(*c)
    inside = torch.zeros(y.shape[0], dtype=torch.bool, device="cuda")
    inside[5:-19] = True
    check(out[inside], c[0][inside], c[1][inside], *c[2:4], offsets - 5, which, s)
    assert torch.equal(out[~inside], c[0][~inside])
    assert torch.equal(ops.lora(*c, out=c[0]), out) and torch.equal(ops.lora(*c[:2], *c[2:], out=torch.empty_like(out)), ops.lora(*c))


@gpu
def test_offsets_that_are_none_with_shared_adapters():
    from ac4k_kernel_b200 import ops
    y, x, a, b, _, adapters, s = case([10] * 6, [0, 1, 0, 1, -1, 0], 64, 48, 8, 2, seed=18)
    big = torch.full((180, 48), 7.0, dtype=y.dtype, device="cuda")
    for bad in ([-5, 10, 20, 30, 40, 50, 60], [0, 10, 20, 1000000, 5, 60, 60], [0, 20, 10, 30, 0, 60, 1], [60, 50, 40, 30, 20, 10, 0],
                [2 ** 31 - 1, -2 ** 31, 2 ** 31 - 1, 5, 2 ** 31 - 1, -7, 60]):
        offsets = torch.tensor(bad, dtype=torch.int32, device="cuda")
        ops.lora(y, x, a, b, offsets, adapters, s, out=big[60:120])
        torch.cuda.synchronize()
        assert bool((big[:60] == 7).all()) and bool((big[120:] == 7).all())


@gpu
@pytest.mark.parametrize("requests", [1, 20000])
def test_rows_past_32_bits(requests):
    """The last rows of x, y and out begin behind 2^32 bytes"""
    from ac4k_kernel_b200 import ops
    t, k, n = 300000, 8192, 8192
    x = torch.randn((t, k), dtype=torch.bfloat16, device="cuda")
    y = torch.randn((t, n), dtype=torch.bfloat16, device="cuda")
    _, _, a, b, _, _, s = case([1], [0], k, n, 16, 2, seed=16)
    offsets = torch.linspace(0, t, requests + 1, dtype=torch.float64).long()
    adapters = torch.arange(requests) % 2
    out = ops.lora(y, x, a, b, offsets.int().cuda(), adapters.int().cuda(), s)
    for lo in (0, t // 2, t - 300):
        which = torch.searchsorted(offsets, torch.arange(lo, lo + 300), right=True) - 1
        rows = slice(lo, lo + 300)
        check(out[rows], y[rows], x[rows], a, b, torch.arange(301), adapters[which], s)


@gpu
def test_many_requests():
    """More requests than threads of a block, most of them empty"""
    from ac4k_kernel_b200 import ops
    g = torch.Generator().manual_seed(1)
    lengths = [int(v) if v > 0 else 0 for v in torch.randint(-6, 4, (1500,), generator=g)]
    c = case(lengths, [i % 9 - 1 for i in range(1500)], 128, 72, 16, 8, lead=3, behind=2, seed=7, scaling=False)
    check(ops.lora(*c), *c)
    c = case([90] * 200, [i % 3 for i in range(200)], 64, 40, 8, 3, seed=8)
    check(ops.lora(*c), *c)


@gpu
def test_nothing_to_do():
    from ac4k_kernel_b200 import ops
    y, x, a, b, offsets, adapters, s = case([4, 4], [0, 1], 64, 48, 8, 2, seed=9)
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    assert torch.equal(ops.lora(y, x, a, b, torch.zeros(1, dtype=torch.int32, device="cuda"), none), y)
    assert torch.equal(ops.lora(y, x, a[:0], b[:0], offsets, adapters), y)
    assert torch.equal(ops.lora(y, x, a[:, :0].contiguous(), b[:, :, :0].contiguous(), offsets, adapters), y)
    assert torch.equal(ops.lora(y, x[:, :0].contiguous(), a[:, :, :0].contiguous(), b, offsets, adapters), y)
    assert ops.lora(y[:0], x[:0], a, b, torch.zeros(3, dtype=torch.int32, device="cuda"), adapters).shape == (0, 48)
    assert ops.lora(y[:, :0].contiguous(), x, a, b[:, :0].contiguous(), offsets, adapters).shape == (8, 0)

@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("t,n", [(8, 48), (8, 45), (1, 48), (200, 2056)])
def test_one_row_of_y_for_all_without_an_adapter(t, n, dtype):
    """Whether y may be one row for all does not hang on whether the batch has adapters, requests, features or a rank"""
    from ac4k_kernel_b200 import ops
    y, x, a, b, offsets, adapters, s = case([t // 2, t - t // 2], [0, 1], 64, n, 8, 2, dtype, seed=22)
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    for rows in (y[:1].expand(t, n), y, torch.cat([y, y], 1)[:, 3:3 + n]):
        want = rows.contiguous()
        big = torch.full((t + 2, n + 24), 7.0, dtype=dtype, device="cuda")
        for out in (None, big[1:-1, 8:8 + n]):
            for call in ((x, a, b, torch.zeros(1, dtype=torch.int32, device="cuda"), none), (x, a[:0], b[:0], offsets, adapters),
                         (x, a[:, :0].contiguous(), b[:, :, :0].contiguous(), offsets, adapters, s),
                         (x[:, :0].contiguous(), a[:, :, :0].contiguous(), b, offsets, adapters, s)):
                got = ops.lora(rows, *call, out=out)
                assert torch.equal(got, want)
                got.fill_(3.0)
        big[1:-1, 8:8 + n] = 7.0
        assert bool((big == 7).all())


@gpu
def test_offsets_that_are_none():
    """Offsets past the rows, negative ones and descending ones reach no memory of others: every row is its own result or y's"""
    from ac4k_kernel_b200 import ops
    y, x, a, b, _, adapters, s = case([10, 10, 10], [0, 1, 0], 64, 48, 8, 2, seed=10)
    big = torch.full((90, 48), 7.0, dtype=y.dtype, device="cuda")
    for bad in ([-5, 10, 20, 30], [0, 10, 20, 1000000], [0, 20, 10, 30], [30, 20, 10, 0], [2 ** 31 - 1, -2 ** 31, 2 ** 31 - 1, 5]):
        offsets = torch.tensor(bad, dtype=torch.int32, device="cuda")
        ops.lora(y, x, a, b, offsets, adapters, s, out=big[30:60])
        torch.cuda.synchronize()
        assert bool((big[:30] == 7).all()) and bool((big[60:] == 7).all())


@gpu
def test_same_result_each_time_streams_and_graphs():
    from ac4k_kernel_b200 import ops
    c = case([1] * 30, [i % 4 for i in range(30)], 2048, 512, 16, 4, seed=11)
    want = ops.lora(*c)
    d = case([700], [0], 1024, 256, 64, 1, seed=12)
    want_d = ops.lora(*d)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(20):
        with torch.cuda.stream(side):
            other = ops.lora(*d)
        assert torch.equal(ops.lora(*c), want)
        side.synchronize()
        assert torch.equal(other, want_d)
    graphs = []
    for args in (c, d):             # two graphs replayed side by side
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = ops.lora(*args)
        graphs.append((graph, out))
    for _ in range(10):
        for _, out in graphs:
            out.zero_()
        torch.cuda.synchronize()
        graphs[0][0].replay()
        with torch.cuda.stream(side):
            graphs[1][0].replay()
        torch.cuda.synchronize()
        assert torch.equal(graphs[0][1], want) and torch.equal(graphs[1][1], want_d)
    c[0].zero_()
    graphs[0][0].replay()
    torch.cuda.synchronize()
    check(graphs[0][1], *c)


@gpu
def test_beside_the_linear_layer():
    """norm -> linear + adapters, in place on the projection's output"""
    from ac4k_kernel_b200 import ops
    _, x, a, b, offsets, adapters, s = case([1, 30, 9], [1, -1, 0], 512, 256, 16, 2, seed=13)
    w4 = ops.quantize(gaussian((256, 512), 3, std=0.05).cuda(), 0, 1)
    q, sf, g, v = ops.rms_norm(x, precision="nvfp4", global_scale=torch.tensor(30 / 2688, device="cuda"), keep=True)
    y = ops.linear(q, sf, g, *w4)
    base = y.clone()
    out = ops.lora(y, v, a, b, offsets, adapters, s, out=y)
    assert out is y
    check(out, base, v, a, b, offsets, adapters, s)


@gpu
def test_native_host_side_and_wrapper_agree(monkeypatch):
    from ac4k_kernel_b200 import ops
    from ac4k_kernel_b200.native import host_calls
    if host_calls is None:
        pytest.skip("the native host side is not built")
    module = sys.modules["ac4k_kernel_b200.ops.lora"]
    y, x, a, b, offsets, adapters, s = case([5, 20], [0, 1], 64, 48, 8, 2, seed=14)
    good = dict(y=y, x=x, a=a, b=b, offsets=offsets, adapters=adapters, scaling=s)
    calls = [dict(), dict(scaling=None), dict(out=torch.empty_like(y)), dict(y=y.half()), dict(y=y.float())]
    wrong = [dict(y=y.double()), dict(y=y[:5]), dict(x=x.float()), dict(x=x[:, :8]), dict(a=a[:1]), dict(b=b[:, :7]), dict(b=b.transpose(1, 2)),
             dict(offsets=offsets[:2]), dict(offsets=offsets.long()), dict(adapters=adapters.long()), dict(scaling=s[:1]), dict(scaling=s.double()),
             dict(out=y.float()), dict(out=y[:5]), dict(y=y.t()), dict(x=x.t()), dict(x=x.cpu()), dict(offsets=offsets.cpu()), dict(y=y.cpu()),
             dict(a=torch.zeros(2, 130, 64, dtype=torch.bfloat16, device="cuda"), b=torch.zeros(2, 48, 130, dtype=torch.bfloat16, device="cuda")),
             dict(out=torch.zeros(26, 48, dtype=torch.bfloat16, device="cuda")[1:, :].as_strided((25, 48), (24, 1)))]
    whole = torch.zeros(26, 48, dtype=torch.bfloat16, device="cuda")
    wrong.append(dict(y=whole[:25], out=whole[1:]))              # overlaps y and is not y
    both = torch.zeros(25, 128, dtype=torch.bfloat16, device="cuda")
    wrong.append(dict(x=both[:, :64], out=both[:, 40:88]))       # overlaps x
    calls.append(dict(x=both[:, :64], out=both[:, 64:112]))      # lies between x's rows
    for number, kw in enumerate(calls + wrong):
        res = []
        for path in (host_calls, None):
            monkeypatch.setattr(module, "host_calls", path)
            try:
                res.append(ops.lora(**{**good, **kw}).clone())
            except Exception as e:
                res.append(type(e))
        if number >= len(calls):
            assert res[0] is res[1] and issubclass(res[0], Exception), (number, res)
        else:
            assert torch.equal(res[0], res[1]), number


def test_refusals_of_the_c_interface():
    """Bad arguments give negative codes before anything touches a device"""
    from ac4k_kernel_b200._lib import LIB, last_error
    P = 1 << 20

    def call(out=P, y=2 * P, dt=0, x=3 * P, a=P, b=P, offsets=P, adapters=P, scaling=None, t=4, s=1, l=1, k=64, n=64, r=8, xs=64, ys=64,
             os=64):
        return LIB.ac4k_lora(out, y, dt, x, a, b, offsets, adapters, scaling, t, s, l, k, n, r, xs, ys, os, None)

    for kw, code in ((dict(dt=3), -4), (dict(t=-1), -2), (dict(r=129), -5), (dict(n=1 << 23), -2), (dict(xs=-1), -2), (dict(out=None), -1),
                     (dict(y=None), -1), (dict(y=2 * P + 1), -3), (dict(y=P + 64), -2), (dict(x=P + 64), -2), (dict(y=P, ys=128), -2), (dict(os=32), -2),
                     (dict(x=None), -1), (dict(offsets=None), -1), (dict(x=P + 1), -3), (dict(adapters=P + 2), -3), (dict(scaling=P + 1), -3),
                     (dict(l=0, ys=8), -2)):
        assert call(**kw) == code, kw
        assert last_error()
    assert call(t=0, out=None) == 0 and call(n=0) == 0
    assert call(out=P, y=P, l=0, x=None) == 0            # in place and nothing to add


def test_one_row_in_place_is_not_refused():
    from ac4k_kernel_b200._lib import LIB
    P = 1 << 20
    for strides in ((64, 64, 64), (64, 128, 64), (64, 64, 7), (1, 0, 0)):
        assert LIB.ac4k_lora(P, P, 0, None, None, None, None, None, None, 1, 0, 0, 64, 64, 8, *strides, None) == 0, strides
    assert LIB.ac4k_lora(P, P, 0, None, None, None, None, None, None, 2, 0, 0, 64, 64, 8, 64, 128, 64, None) == -2
