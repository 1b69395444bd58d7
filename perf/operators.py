"""What the operators around the NVFP4 linear layer are measured on: `rms_norm` in front of it, `lora` beside it, `linear_grouped`
in its place.

  norm      the residual's addition and the RMS norm of the hidden states, in bf16 or in e4m3 with one scale a row
  lora      the low-rank adapters of a batch of requests, added to the output of the projection that all of them share
  grouped   a linear layer with a weight per expert, on rows that are sorted by expert: NVFP4 operands, ragged groups
  block     the three calls of a projection with adapters: norm to NVFP4 -> `linear` -> adapters

`own` false: the operators in plain form, elementary torch operations in fp32, rounded once at the end.  `own` true: the calls of
`ac4k_kernel_b200.ops` that a program makes.
"""
import math

import torch

own = False

_EPS = 1e-6
_MAX_ROWS = 32768 * 8192                   # elements of the largest tensor that is normalised
_MAX_LORA = 8192 * (8192 + 2 * 8192)       # T * (K + 2 N) of the largest adapter call
_MAX_EXPERTS = 1 << 28                     # E * N * K of the largest stack of experts' weights
_MAX_GROUPED = 16384 * 8192 * 4096         # T * N * K of the largest grouped product
_E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0]


def _norm(name, rows, cols, out, residual=True):
    return {"name": name, "kind": "norm", "rows": rows, "cols": cols, "out": out, "residual": residual}


def _lora(name, requests, tokens, k, n, rank, adapters, without=0, out="bf16"):
    return {"name": name, "kind": "lora", "requests": requests, "tokens": tokens, "k": k, "n": n, "rank": rank, "adapters": adapters,
            "without": without, "out": out}


def _grouped(name, experts, tokens, k, n, idle=0, bias=False, out="bf16"):
    return {"name": name, "kind": "grouped", "experts": experts, "tokens": tokens, "k": k, "n": n, "idle": idle, "bias": bias, "out": out}


def _block(name, requests, tokens, k, n, rank, adapters):
    return {"name": name, "kind": "block", "requests": requests, "tokens": tokens, "k": k, "n": n, "rank": rank, "adapters": adapters}


def listed():
    return [
        # one token of one sequence: launches and one row's two reductions
        _norm("norm_fp8_1", 1, 8192, "fp8e4m3"),
        # a prompt batch with an odd number of rows
        _norm("norm_fp8_4099", 4099, 5120, "fp8e4m3"),
        # the norm in front of a layer that stays in bf16, no residual (the first norm of a model)
        _norm("norm_bf16_666", 666, 4096, "bf16", residual=False),
        # a large prefill: the largest tensor
        _norm("norm_fp8_32768", 32768, 8192, "fp8e4m3"),
        # a decode batch, one token each, every request with an adapter of its own: the adapters' bytes
        _lora("lora_decode_64", 64, 64, 8192, 8192, 16, 64),
        # prompts of ragged lengths, some requests without an adapter
        _lora("lora_ragged_4099", 9, 4099, 4096, 4096, 64, 5, without=4),
        # a long prompt through one adapter
        _lora("lora_8192", 1, 8192, 8192, 8192, 32, 1),
        # one token, two experts of many: the smallest product
        _grouped("grouped_decode_2", 64, 2, 4096, 1024),
        # a decode batch over few large experts: the stream of all their weights
        _grouped("grouped_decode_32", 8, 32, 4096, 8192, bias=True),
        # a prompt over many experts, uneven, a quarter of them without a row
        _grouped("grouped_ragged_4099", 64, 4099, 2048, 2048, idle=4),
        # a large prefill over few experts: the tensor pipe
        _grouped("grouped_16384", 8, 16384, 4096, 8192),
        # a decode batch through a projection with adapters, norm included
        _block("block_50", 50, 50, 8192, 8192, 16, 8),
    ]


def _log(rng, lo, hi):
    """An integer of [lo, hi], even over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _to(x, multiple):
    return max(multiple, x // multiple * multiple)


def draw(rng):
    kind = rng.choices(["norm", "lora", "grouped", "block"], [3, 4, 4, 1])[0]
    if kind == "norm":
        # features: multiples of 64 as layers have them, now and then odd
        cols = _to(_log(rng, 256, 16384), rng.choice([64, 64, 64, 8, 1]))
        rows = min(_log(rng, 1, 32768), _MAX_ROWS // cols)
        return {"kind": kind, "rows": rows, "cols": cols, "out": rng.choice(["fp8e4m3", "fp8e4m3", "bf16"]), "residual": rng.random() < 0.8}
    if kind == "lora":
        requests = _log(rng, 1, 128)
        tokens = requests if rng.random() < 0.5 else max(requests, _log(rng, 1, 8192))
        k, n = (_to(_log(rng, 512, 8192), rng.choice([64, 64, 64, 8])) for _ in range(2))
        while tokens > requests and tokens * (k + 2 * n) > _MAX_LORA:
            tokens = max(requests, tokens // 2)
        return {"kind": kind, "requests": requests, "tokens": tokens, "k": k, "n": n, "rank": rng.choice([4, 8, 16, 16, 32, 64, 128]),
                "adapters": rng.choice([1, 4, 16, 64]), "without": rng.choice([0, 0, 2, 5]), "out": rng.choices(["bf16", "fp16", "fp32"], [6, 1, 1])[0]}
    if kind == "grouped":
        experts = rng.choice([4, 8, 16, 32, 64, 128])
        n, k = _to(_log(rng, 256, 8192), rng.choice([64, 64, 8])), _to(_log(rng, 256, 8192), 64)
        while experts * n * k > _MAX_EXPERTS:
            n, k = _to(n // 2, 8), _to(k // 2, 64)
        tokens = _log(rng, 1, 16384)
        while tokens * n * k > _MAX_GROUPED:
            tokens //= 2
        return {"kind": kind, "experts": experts, "tokens": tokens, "k": k, "n": n, "idle": rng.choice([0, 0, 2, 4]), "bias": rng.random() < 0.3,
                "out": rng.choices(["bf16", "fp16", "fp32"], [6, 1, 1])[0]}
    requests = _log(rng, 1, 64)
    tokens = requests if rng.random() < 0.5 else max(requests, _log(rng, 1, 4096))
    k, n = (_to(_log(rng, 512, 8192), 64) for _ in range(2))
    return {"kind": kind, "requests": requests, "tokens": tokens, "k": k, "n": n, "rank": rng.choice([8, 16, 32, 64]),
            "adapters": rng.choice([1, 4, 8])}


# ---- inputs -------------------------------------------------------------------------------------
_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _activations(shape, g):
    """N(0, 1) with half a percent of outliers thirty times as large, as hidden states have them."""
    x = torch.randn(shape, generator=g, device="cuda", dtype=torch.bfloat16)
    return torch.where(torch.rand(shape, generator=g, device="cuda", dtype=torch.float16) < 0.005, x * 30, x)


def _lengths(total, parts, seed, used=None):
    """Uneven lengths of `parts` groups that add up to `total`, at least one for each group that is used (as far as `total` goes)."""
    g = torch.Generator().manual_seed(seed + 1)
    order = torch.randperm(parts, generator=g)[:min(parts if used is None else used, total)]
    share = torch.rand(len(order), generator=g, dtype=torch.float64) ** 2 + 0.05
    n = 1 + ((total - len(order)) * share / share.sum()).floor().long()
    n[0] += total - int(n.sum())
    lengths = torch.zeros(parts, dtype=torch.long)
    lengths[order] = n
    return lengths


def _offsets(lengths):
    return torch.cat([torch.zeros(1, dtype=torch.long), lengths.cumsum(0)])


def _adapter_of(case):
    """Adapter of each request: in turn, every `without`-th request none."""
    without = case.get("without", 0)
    return [-1 if without and i % without == without - 1 else i % case["adapters"] for i in range(case["requests"])]


def _used_experts(case):
    idle = case["experts"] // case["idle"] if case["idle"] else 0
    return min(case["experts"] - idle, case["tokens"])


def _e4m3(x):
    return x.clamp(-448.0, 448.0).to(torch.float8_e4m3fn)


def _to_nvfp4(x, global_scale):
    """fp32 [.., M, K], K a multiple of 64 -> packed e2m1 [.., M, K / 2], e4m3 scales [.., K / 64, M to 16, 4] of blocks of 16 along K.
    A scale is the block's maximum over 6 in units of the global scale; ties of a code go to the even one."""
    lead, (m, k) = x.shape[:-2], x.shape[-2:]
    alpha = 1.0 / global_scale
    blocks = x.reshape(*lead, m, k // 16, 16)
    sf = _e4m3(blocks.abs().amax(-1) * (1.0 / 6.0) * alpha)
    back = sf.float()
    r = torch.where(back > 0, alpha / back, torch.zeros_like(back))
    y = blocks * r.unsqueeze(-1)
    a = y.abs()
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0)).to(torch.uint8)
    code = (code | (torch.signbit(y).to(torch.uint8) << 3)).reshape(*lead, m, k // 2, 2)
    packed = code[..., 0] | (code[..., 1] << 4)
    rows = torch.zeros(*lead, k // 64, (m + 15) // 16 * 16, 4, dtype=torch.uint8, device=x.device)
    rows[..., :m, :] = sf.view(torch.uint8).reshape(*lead, m, k // 64, 4).transpose(-3, -2)
    return packed, rows.view(torch.float8_e4m3fn)


def _from_nvfp4(packed, sf, dtype):
    """The values that packed codes and block scales stand for, without the global scale: [.., M, K]."""
    lead, (m, half) = packed.shape[:-2], packed.shape[-2:]
    lut = torch.tensor(_E2M1, dtype=dtype, device=packed.device)
    values = torch.stack((lut[(packed & 15).int()], lut[(packed >> 4).int()]), -1).reshape(*lead, m, half // 8, 16)
    scales = sf.to(dtype)[..., :m, :].transpose(-3, -2).reshape(*lead, m, half // 8)
    return (values * scales.unsqueeze(-1)).reshape(*lead, m, half * 2)


def _quantised(x):
    """A bf16 tensor as `quantize` leaves it: codes, block scales, the global scale that takes the largest value to 6 x 448."""
    x = x.float()
    g = x.abs().max() / (448.0 * 6.0)
    return (*_to_nvfp4(x, g), g)


def prepare(case, seed):
    g = _generator(seed)
    kind = case["kind"]
    if kind == "norm":
        shape = (case["rows"], case["cols"])
        s = {"x": _activations(shape, g), "weight": (1 + 0.2 * torch.randn(case["cols"], generator=g, device="cuda")).bfloat16()}
        if case["residual"]:
            s["residual"] = _activations(shape, g)
    elif kind == "grouped":
        e, t, k, n = case["experts"], case["tokens"], case["k"], case["n"]
        lengths = _lengths(t, e, seed, _used_experts(case))
        s = {"offsets": _offsets(lengths).int().cuda(), "longest": int(lengths.max())}
        s["x"] = _quantised(_activations((t, k), g))
        s["w"] = _quantised(torch.randn((e, n, k), generator=g, device="cuda", dtype=torch.bfloat16) * 0.02)
        s["bias"] = torch.randn((e, n), generator=g, device="cuda", dtype=torch.bfloat16) if case["bias"] else None
    else:
        r, t, k, n, a = case["requests"], case["tokens"], case["k"], case["n"], case["adapters"]
        lengths = _lengths(t, r, seed)
        s = {"offsets": _offsets(lengths).int().cuda(), "longest": int(lengths.max())}
        s["adapters"] = torch.tensor(_adapter_of(case), dtype=torch.int32, device="cuda")
        s["a"] = torch.randn((a, case["rank"], k), generator=g, device="cuda", dtype=torch.bfloat16) * k ** -0.5
        s["b"] = torch.randn((a, n, case["rank"]), generator=g, device="cuda", dtype=torch.bfloat16) * 0.1
        s["scaling"] = 0.5 + torch.rand(a, generator=g, device="cuda")
        s["x"] = _activations((t, k), g)
        if kind == "lora":
            s["y"] = torch.randn((t, n), generator=g, device="cuda").to(_DTYPES[case["out"]])
        else:
            s["residual"] = _activations((t, k), g)
            s["weight"] = (1 + 0.2 * torch.randn(k, generator=g, device="cuda")).bfloat16()
            s["w"] = _quantised(torch.randn((n, k), generator=g, device="cuda", dtype=torch.bfloat16) * 0.02)
            # as calibration finds it: normalised hidden states reach some thirty times their root mean square
            s["global_scale"] = torch.tensor(40.0 / (448.0 * 6.0), device="cuda")
    s["case"] = dict(case)
    return s


# ---- the plain forms ----------------------------------------------------------------------------
def _normed(x, residual, weight):
    s = x.float()
    if residual is not None:
        s = s + residual.float()
    v = s * torch.rsqrt((s * s).mean(-1, keepdim=True) + _EPS) * weight.float()
    return s, v


def _padded_rows(offsets, longest, total):
    """Row of each place in a [groups, longest] table, clamped; and of each row its group and its place there."""
    first, last = offsets[:-1].long(), offsets[1:].long()
    rows = (first[:, None] + torch.arange(longest, device=offsets.device)).clamp(max=total - 1)
    t = torch.arange(total, device=offsets.device)
    group = torch.searchsorted(last, t, right=True)
    return rows, group, t - first[group]


def _plain_lora(y, x, s):
    rows, group, place = _padded_rows(s["offsets"], s["longest"], x.shape[0])
    which = s["adapters"].clamp(min=0).long()
    low = torch.bmm(x.float()[rows], s["a"].float()[which].transpose(1, 2))
    delta = torch.bmm(low, s["b"].float()[which].transpose(1, 2)) * (s["scaling"][which] * (s["adapters"] >= 0))[:, None, None]
    return y.float() + delta[group, place]


def _plain(s):
    case = s["case"]
    kind = case["kind"]
    if kind == "norm":
        total, v = _normed(s["x"], s.get("residual"), s["weight"])
        extra = [total.bfloat16()] if case["residual"] else []
        if case["out"] == "bf16":
            return [v.bfloat16(), *extra]
        m, k = v.shape
        scale = v.abs().amax(-1) / 448.0
        codes = torch.zeros(m, (k + 15) // 16 * 16, dtype=torch.float8_e4m3fn, device=v.device)
        codes[:, :k] = _e4m3(v / scale[:, None])
        sf = torch.zeros((m + 15) // 16 * 16, device=v.device)
        sf[:m] = scale
        return [codes, sf, *extra]
    if kind == "lora":
        return [_plain_lora(s["y"], s["x"], s).to(s["y"].dtype)]
    if kind == "grouped":
        (xq, xsf, xg), (wq, wsf, wg) = s["x"], s["w"]
        x, w = _from_nvfp4(xq, xsf, torch.float32), _from_nvfp4(wq, wsf, torch.float32)
        rows, group, place = _padded_rows(s["offsets"], s["longest"], x.shape[0])
        y = torch.bmm(x[rows], w.transpose(1, 2)) * (xg * wg)
        if s["bias"] is not None:
            y = y + s["bias"].float()[:, None, :]
        return [y[group, place].to(_DTYPES[case["out"]])]
    total, v = _normed(s["x"], s["residual"], s["weight"])
    wq, wsf, wg = s["w"]
    x = _from_nvfp4(*_to_nvfp4(v, s["global_scale"]), torch.float32)
    y = x @ _from_nvfp4(wq, wsf, torch.float32).t() * (s["global_scale"] * wg)
    return [_plain_lora(y, v.bfloat16(), s).bfloat16(), total.bfloat16()]


# ---- the calls of a program ---------------------------------------------------------------------
def _calls(s):
    from ac4k_kernel_b200 import ops
    case = s["case"]
    kind = case["kind"]
    if kind == "norm":
        r = ops.rms_norm(s["x"], s["weight"], _EPS, residual=s.get("residual"), precision=None if case["out"] == "bf16" else case["out"])
        return list(r) if isinstance(r, tuple) else [r]
    if kind == "lora":
        return [ops.lora(s["y"], s["x"], s["a"], s["b"], s["offsets"], s["adapters"], s["scaling"])]
    if kind == "grouped":
        out = None if case["out"] == "bf16" else torch.empty((case["tokens"], case["n"]), dtype=_DTYPES[case["out"]], device="cuda")
        return [ops.linear_grouped(*s["x"], *s["w"], s["offsets"], bias=s["bias"], out=out)]
    q, sf, gs, v, total = ops.rms_norm(s["x"], s["weight"], _EPS, residual=s["residual"], precision="nvfp4", global_scale=s["global_scale"], keep=True)
    y = ops.linear(q, sf, gs, *s["w"])
    return [ops.lora(y, v, s["a"], s["b"], s["offsets"], s["adapters"], s["scaling"], out=y), total]


def run(state):
    return _calls(state) if own else _plain(state)


# ---- bytes and operations -----------------------------------------------------------------------
def work(case):
    kind = case["kind"]
    if kind == "norm":
        m, k = case["rows"], case["cols"]
        return {"bytes": m * k * (2 + (4 if case["residual"] else 0) + (2 if case["out"] == "bf16" else 1)) + 2 * k + 4 * m, "flops": 8 * m * k}
    if kind == "grouped":
        t, k, n = case["tokens"], case["k"], case["n"]
        out = 4 if case["out"] == "fp32" else 2
        return {"bytes": t * k * 9 / 16 + _used_experts(case) * n * k * 9 / 16 + t * n * out, "flops": 2 * t * n * k}
    t, k, n, rank = case["tokens"], case["k"], case["n"], case["rank"]
    used = len({a for a in _adapter_of(case) if a >= 0})
    weights = used * rank * (k + n) * 2
    out = 4 if case.get("out") == "fp32" else 2
    if kind == "lora":
        return {"bytes": t * k * 2 + 2 * t * n * out + weights, "flops": 2 * t * rank * (k + n)}
    return {"bytes": t * k * 6 + n * k * 9 / 16 + t * n * 2 + weights, "flops": 2 * t * n * k + 2 * t * rank * (k + n)}


# ---- the results in 64 bits ---------------------------------------------------------------------
def _round_e4m3(v):
    """Nearest value of e4m3 (ties to even, at most 448), in float64."""
    step = torch.ldexp(torch.ones_like(v), torch.frexp(v.abs().clamp(min=2.0 ** -6))[1] - 4)
    return (torch.round(v / step) * step).clamp(-448.0, 448.0)


def _round_e2m1(v):
    step = torch.ldexp(torch.ones_like(v), torch.frexp(v.abs().clamp(min=1.0))[1] - 2)
    return (torch.round(v / step) * step).clamp(-6.0, 6.0)


def _exact_norm(x, residual, weight):
    total = x.double() if residual is None else x.double() + residual.double()
    return total, total / (total.square().mean(1, keepdim=True) + _EPS).sqrt() * weight.double()


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]

    def with_adapters(y, x):
        out = y.double().clone()
        bounds = _offsets(_lengths(case["tokens"], case["requests"], seed)).tolist()
        for i, a in enumerate(_adapter_of(case)):
            lo, hi = bounds[i], bounds[i + 1]
            if a >= 0 and hi > lo:
                out[lo:hi] += s["scaling"][a].double() * ((x[lo:hi].double() @ s["a"][a].double().t()) @ s["b"][a].double().t())
        return out

    if kind == "norm":
        total, v = _exact_norm(s["x"], s.get("residual"), s["weight"])
        extra = [total] if case["residual"] else []
        if case["out"] == "bf16":
            return [v, *extra]
        m, k = v.shape
        scale = v.abs().amax(1) / 448
        codes, sf = v.new_zeros(m, -(-k // 16) * 16), v.new_zeros(-(-m // 16) * 16)
        codes[:, :k], sf[:m] = _round_e4m3(v / scale[:, None]), scale
        return [codes, sf, *extra]
    if kind == "lora":
        return [with_adapters(s["y"], s["x"])]
    if kind == "grouped":
        (xq, xsf, xg), (wq, wsf, wg) = s["x"], s["w"]
        x = _from_nvfp4(xq, xsf, torch.float64) * xg.double()
        out = x.new_zeros(case["tokens"], case["n"])
        bounds = _offsets(_lengths(case["tokens"], case["experts"], seed, _used_experts(case))).tolist()
        for e in range(case["experts"]):
            lo, hi = bounds[e], bounds[e + 1]
            if hi > lo:
                out[lo:hi] = x[lo:hi] @ (_from_nvfp4(wq[e], wsf[e], torch.float64) * wg.double()).t()
                if s["bias"] is not None:
                    out[lo:hi] += s["bias"][e].double()
        return [out]
    total, v = _exact_norm(s["x"], s["residual"], s["weight"])
    m, k = v.shape
    g = s["global_scale"].double()
    blocks = v.reshape(m, k // 16, 16)
    sf = _round_e4m3(blocks.abs().amax(2) / 6 / g) * g
    x = (_round_e2m1(blocks / sf[:, :, None].clamp(min=1e-300)) * sf[:, :, None]).reshape(m, k)
    wq, wsf, wg = s["w"]
    y = x @ (_from_nvfp4(wq, wsf, torch.float64) * wg.double()).t()
    return [with_adapters(y, v.bfloat16()), total]
