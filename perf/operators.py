"""Workloads of the MXFP8 serving path: the operators from the norm before a linear layer to its product.

    norm    residual addition, RMSNorm and MXFP8 codes with scales    vllm_qdq_plugin.qdq.rmsnorm_mxfp8
    gate    SiLU-gated product and MXFP8 codes with scales            vllm_qdq_plugin.qdq.silu_mul_mxfp8
    linear  dense product of MXFP8 rows and an MXFP8 weight           vllm_qdq_plugin.gemm.mxfp8_linear
    moe     the same product grouped by expert, ragged                vllm_qdq_plugin.gemm.mxfp8_moe_linear

MXFP8: E4M3 codes, one E8M0 scale 2^e per 32 consecutive elements of a row, e = floor(log2 amax) - 8, codes rounded to nearest even and
saturated at 448; below 2^-6 (E4M3's subnormals) the rounded magnitude is at most 7 * 2^-9, as in the framework's mxfp8_qdq.

With `own` false every operator runs in its plain form, elementary torch operations on 32-bit values (the norm in 64: its output is
rounded twice, and values next to a border decide a code); with `own` true it runs as the framework's call.
"""

import math
import sys

import numpy as np
import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
_EPS = 1e-6


def _package():
    if "vllm-qdq-plugin_b200" not in sys.path:
        sys.path.insert(0, "vllm-qdq-plugin_b200")
    from vllm_qdq_plugin import gemm, qdq
    return qdq, gemm


# ---------------------------------------------------------------------------- cases
def _norm(name, m, k, dtype="bf16", residual=True, norm_out=False):
    return dict(name=name, op="norm", m=m, k=k, dtype=dtype, residual=residual, norm_out=norm_out)


def _gate(name, m, k, dtype="bf16"):
    return dict(name=name, op="gate", m=m, k=k, dtype=dtype)


def _linear(name, m, n, k, dtype="bf16", codes=False, bias=False):
    return dict(name=name, op="linear", m=m, n=n, k=k, dtype=dtype, codes=codes, bias=bias)


def _moe(name, m, e, top_k, n, k, block, dtype="bf16", codes=False, mul=False):
    return dict(name=name, op="moe", m=m, e=e, top_k=top_k, n=n, k=k, block=block, dtype=dtype, codes=codes, mul=mul)


def listed():
    return [
        # one token of a decode step in front of a hidden-4096 layer: latency alone
        _norm("norm one token", 1, 4096),
        # a ragged batch of prompts in fp16, hidden 2880, the 16-bit norm kept for a router
        _norm("norm ragged routed", 777, 2880, "fp16", norm_out=True),
        # a long prefill at hidden 8192: HBM traffic
        _norm("norm prefill", 16384, 8192),
        # 64 decoded tokens, top-4: the rows between the experts' two products
        _gate("gate decode slots", 256, 2880),
        # a 4096-token prefill of a dense layer with intermediate size 14336
        _gate("gate prefill", 4096, 14336, "fp16"),
        # one token against a square attention projection: the smallest product
        _linear("linear one token", 1, 4096, 4096),
        # a decode batch against an MLP projection: the weight's bytes
        _linear("linear decode batch", 16, 14336, 4096),
        # a short ragged prompt, odd sizes, bias, fp16, rows that a norm already left in 8 bits
        _linear("linear ragged bias", 333, 1001, 2880, "fp16", codes=True, bias=True),
        # the same MLP projection in a 4096-token prefill, from the norm's codes: tensor cores
        _linear("linear prefill", 4096, 14336, 4096, codes=True),
        # one token through a small expert layer's first product
        _moe("experts one token", 1, 32, 4, 2880, 2880, 16),
        # 64 decoded tokens over 128 experts, top-4, from the norm's codes: the hit experts' bytes
        _moe("experts decode", 64, 128, 4, 5760, 2880, 16, codes=True, mul=True),
        # a 4096-token prefill over the same layer
        _moe("experts prefill", 4096, 128, 4, 5760, 2880, 64),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "gate", "linear", "moe"])
    dtype = rng.choice(["bf16", "fp16"])
    if op == "norm":
        k = 32 * _log(rng, 2, 256)
        m = _log(rng, 1, min(16384, 16384 * 8192 // k))
        c = _norm("", m, k, dtype, rng.random() < 0.7, rng.random() < 0.3)
    elif op == "gate":
        k = 32 * _log(rng, 2, 448)
        m = _log(rng, 1, min(16384, 4096 * 14336 // k))
        c = _gate("", m, k, dtype)
    elif op == "linear":
        k, n = 32 * _log(rng, 4, 256), _log(rng, 64, 14336)
        m = _log(rng, 1, min(4096, 4096 * 14336 * 4096 // (n * k)))
        c = _linear("", m, n, k, dtype, rng.random() < 0.5, rng.random() < 0.5)
    else:
        e = rng.choice([4, 8, 16, 32, 64, 128])
        k, n = 32 * _log(rng, 4, 90), _log(rng, 64, 5760)
        top_k, block = rng.choice([1, 2, 4]), rng.choice([8, 16, 32, 48, 64])
        c = _moe("", _log(rng, 1, 4096), e, top_k, n, k, block, dtype, rng.random() < 0.5, rng.random() < 0.5)
    del c["name"]
    return c


# ---------------------------------------------------------------------------- inputs
def _quantised(x):
    """Row-major E4M3 codes (float8) and E8M0 bytes of 16-bit rows: what a layer before left in 8 bits."""
    m, k = x.shape
    g = x.float().view(m, k // 32, 32)
    e = torch.frexp(g.abs().amax(-1).clamp_min(2.0 ** -126))[1] - 9
    q = torch.ldexp(g, -e[..., None]).clamp(-448, 448)
    q = torch.where((q.abs() >= 7 * 2.0 ** -9) & (q.abs() < 2.0 ** -6), torch.copysign(torch.full_like(q, 7 * 2.0 ** -9), q), q)
    return q.view(m, k).to(torch.float8_e4m3fn), (e + 127).to(torch.uint8)


def _weight(shape, g, dev):
    """E4M3 codes spread as a quantised weight's and E8M0 scales around 2^-11."""
    codes = torch.randn(shape, generator=g, device=dev, dtype=torch.bfloat16).mul_(110).clamp_(-448, 448).to(torch.float8_e4m3fn)
    scales = torch.randint(114, 119, (*shape[:-1], shape[-1] // 32), generator=g, device=dev, dtype=torch.uint8)
    return codes, scales


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dtype = _DTYPES[case["dtype"]]
    m, k = case["m"], case["k"]
    s = {"case": case, "dtype": dtype}

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    if case["op"] == "norm":
        s["x"] = normal(m, k).to(dtype)
        s["w"] = (1 + 0.1 * normal(k)).to(dtype)
        # the residual stream grows over a model's depth
        s["residual"] = (normal(m, k) * 4).to(dtype) if case["residual"] else None
        return s
    if case["op"] == "gate":
        s["x"] = (normal(m, 2 * k) * 2).to(dtype)
        return s
    # normed rows with a few strong channels
    x = (normal(m, k) * (1 + 9 * (torch.rand(k, generator=g, device=dev) < 0.01))).to(dtype)
    if case["codes"]:
        s["a_codes"], s["a_scales"] = _quantised(x)
    else:
        s["x"] = x
    if case["op"] == "linear":
        s["w_codes"], s["w_scales"] = _weight((case["n"], k), g, dev)
        s["bias"] = normal(case["n"]).to(dtype) if case["bias"] else None
    else:
        e, top_k, block = case["e"], case["top_k"], case["block"]
        s["w_codes"], s["w_scales"] = _weight((e, case["n"], k), g, dev)
        # routing: top_k distinct experts a token, slots sorted by expert, each expert's run padded to whole blocks
        ids = torch.rand(m, e, generator=g, device=dev).argsort(1)[:, :top_k].reshape(-1).cpu().numpy()
        counts = np.bincount(ids, minlength=e)
        padded = (counts + block - 1) // block * block
        order = np.argsort(ids, kind="stable")
        rank = np.empty_like(ids)
        rank[order] = np.arange(ids.size) - np.repeat(np.cumsum(counts) - counts, counts)
        sorted_ids = np.full(int(padded.sum()), m * top_k, np.int32)
        sorted_ids[(np.cumsum(padded) - padded)[ids] + rank] = np.arange(ids.size)
        s["ids"], s["rank"], s["cap"] = torch.from_numpy(ids).to(dev), torch.from_numpy(rank).to(dev), int(counts.max())
        s["sorted"] = torch.from_numpy(sorted_ids).to(dev)
        s["experts"] = torch.from_numpy(np.repeat(np.arange(e, dtype=np.int32), padded // block)).to(dev)
        s["padded"] = torch.tensor([sorted_ids.size], dtype=torch.int32, device=dev)
        s["topk_w"] = torch.rand(m, top_k, generator=g, device=dev)
    if own:  # the layouts that a server keeps: the weight's, and the rows' that the layer before hands over
        qdq, gemm = _package()
        lay = gemm.prepare_mxfp8_weight if case["op"] == "linear" else gemm.prepare_mxfp8_moe_weight
        s["weight"] = lay(s["w_codes"].view(torch.uint8), s["w_scales"])
        if case["codes"]:
            s["x"] = qdq.Mxfp8Rows.from_codes(s["a_codes"].view(torch.uint8), s["a_scales"], dtype)
    return s


# ---------------------------------------------------------------------------- plain forms
def _mxfp8(v):
    """E4M3 values and scales 2^e of rows of 16-bit values, in 32 bits."""
    m, k = v.shape
    g = v.float().view(m, k // 32, 32)
    e = torch.floor(torch.log2(g.abs().amax(-1, keepdim=True).clamp_min(2.0 ** -126))).clamp_min(-119) - 8
    mag = (g.abs() * torch.exp2(-e)).clamp_max(448.0)
    step = torch.exp2(torch.floor(torch.log2(mag.clamp_min(2.0 ** -6))) - 3)
    r = torch.round(mag / step) * step
    r = torch.where(mag < 2.0 ** -6, r.clamp_max(7 * 2.0 ** -9), r)
    return (torch.sign(g) * r).view(m, k), torch.exp2(e).view(m, k // 32)


def _rows_of(codes, scales):
    """The values that E4M3 codes and E8M0 bytes stand for, in 32 bits."""
    v = codes.float().view(*scales.shape, 32) * torch.exp2(scales.float() - 127).unsqueeze(-1)
    return v.view(codes.shape)


def _activation(s):
    if s["case"]["codes"]:
        return _rows_of(s["a_codes"], s["a_scales"])
    v, sc = _mxfp8(s["x"])
    return (v.view(*sc.shape, 32) * sc.unsqueeze(-1)).view(v.shape)


def _codes_out(v):
    codes, scales = _mxfp8(v)
    return {"codes": codes.to(torch.float8_e4m3fn), "scales": scales.to(torch.float8_e8m0fnu)}


def _plain(s):
    c, dtype = s["case"], s["dtype"]
    if c["op"] == "norm":
        h = s["x"].float()
        if c["residual"]:
            h = h + s["residual"].float()
        h = h.to(dtype)
        d = h.double()
        y = (d * torch.rsqrt(d.square().mean(1, keepdim=True) + _EPS) * s["w"].double()).to(dtype)
        out = _codes_out(y)
        if c["residual"]:
            out["residual"] = h
        if c["norm_out"]:
            out["norm"] = y
        return out
    if c["op"] == "gate":
        g, u = s["x"].float().chunk(2, 1)
        return _codes_out((g / (1 + torch.exp(-g)) * u).to(dtype))
    a = _activation(s)
    if c["op"] == "linear":
        y = a @ _rows_of(s["w_codes"], s["w_scales"]).t()
        return (y if s["bias"] is None else y + s["bias"].float()).to(dtype)
    # every expert's rows in a slab of its own, as many as the busiest has
    slot = torch.arange(s["ids"].numel(), device=a.device)
    slab = a.new_zeros(c["e"], s["cap"], c["k"])
    slab[s["ids"], s["rank"]] = a[slot // c["top_k"]]
    y = torch.bmm(slab, _rows_of(s["w_codes"], s["w_scales"]).transpose(1, 2))[s["ids"], s["rank"]]
    return (y * s["topk_w"].view(-1, 1) if c["mul"] else y).to(dtype)


def _own(s):
    qdq, gemm = _package()
    c = s["case"]
    if c["op"] == "norm":
        rows, h, y = qdq.rmsnorm_mxfp8(s["x"], s["w"], s["residual"], _EPS, norm_out=c["norm_out"])
    elif c["op"] == "gate":
        rows, h, y = qdq.silu_mul_mxfp8(s["x"]), None, None
    elif c["op"] == "linear":
        return gemm.mxfp8_linear(s["x"], s["weight"], s["bias"])
    else:
        return gemm.mxfp8_moe_linear(s["x"], s["weight"], s["sorted"], s["experts"], s["padded"], s["topk_w"], c["block"], c["top_k"], c["mul"])
    out = {"codes": rows.codes.view(torch.float8_e4m3fn), "scales": rows.scales.view(torch.float8_e8m0fnu)}
    if h is not None:
        out["residual"] = h
    if y is not None:
        out["norm"] = y
    return out


def run(state):
    return _own(state) if own else _plain(state)


# ---------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    m, k = case["m"], case["k"]
    codes = m * k + m * k // 32
    if case["op"] == "norm":
        each = 2 + (4 if case["residual"] else 0) + (2 if case["norm_out"] else 0)
        return {"bytes": m * k * each + codes + 2 * k, "flops": 8 * m * k}
    if case["op"] == "gate":
        return {"bytes": 4 * m * k + codes, "flops": 8 * m * k}
    rows, n = codes if case["codes"] else 2 * m * k, case["n"]
    matrix = n * k + n * k // 32
    if case["op"] == "linear":
        return {"bytes": rows + matrix + 2 * m * n + (2 * n if case["bias"] else 0), "flops": 2 * m * n * k}
    hit = case["e"] * (1 - (1 - case["top_k"] / case["e"]) ** m)  # experts with a token, on average
    slots = m * case["top_k"]
    return {"bytes": rows + hit * matrix + 2 * slots * n + 4 * slots * (2 if case["mul"] else 1), "flops": 2 * slots * n * k}


# ---------------------------------------------------------------------------- from the definition, in 64 bits
def _exact_rows(s):
    if s["case"]["codes"]:
        codes, scales = s["a_codes"], s["a_scales"]
    else:
        codes, scales = _quantised(s["x"])
    return _exact_values(codes, scales)


def _exact_values(codes, scales):
    return torch.ldexp(codes.double(), (scales.int() - 127).repeat_interleave(32, -1))


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        h = s["x"].double() + (s["residual"].double() if case["residual"] else 0)
        stored = h.to(s["dtype"]).double()  # the norm reads the residual stream as it is stored
        y = stored / (stored.pow(2).sum(1, keepdim=True) / case["k"] + _EPS).sqrt() * s["w"].double()
        # codes and scales are roundings of a rounded value: no value in 64 bits stands for them
        out = {"codes": None, "scales": None}
        if case["residual"]:
            out["residual"] = h
        if case["norm_out"]:
            out["norm"] = y
        return out
    if case["op"] == "gate":
        return None
    a = _exact_rows(s)
    if case["op"] == "linear":
        y = torch.einsum("mk,nk->mn", a, _exact_values(s["w_codes"], s["w_scales"]))
        return y if s["bias"] is None else y + s["bias"].double()
    ids = s["ids"].cpu()
    y = torch.empty(ids.numel(), case["n"], dtype=torch.float64, device=a.device)
    for e in range(case["e"]):
        at = torch.nonzero(ids == e)[:, 0].to(a.device)
        if at.numel():
            y[at] = a[at // case["top_k"]] @ _exact_values(s["w_codes"][e], s["w_scales"][e]).t()
    return y * s["topk_w"].double().view(-1, 1) if case["mul"] else y
