"""What is measured of the single-token and norm operators: cases, plain forms, calls.

Operators (nvfp4_b200): ``norm.rms_norm_fp8`` / ``norm.rms_norm_nvfp4`` (residual
addition, root-mean-square norm, quantised output), ``gemv.gemv`` and
``gemv.dual_gemv`` (a few tokens times NVFP4 weights, plain and SiLU-gated) and
``moe.gemv`` / ``moe.dual_gemv`` (the same with each token's chosen experts).

Weights are in the framework's NVFP4 layout: e2m1 codes two per byte [N, K/2]
(element 2i in the low nibble) and one e4m3 scale per 16 columns in 512-byte
atoms [ceil(N/128)][K/64][32][4][4], byte (r%32, (r%128)//32, k%4) of atom
(r//128, k//4) being the scale of row r, block k.
"""
import math
import sys

import torch

own = False

EPS = 1e-6
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def listed():
    return [
        # one decoded token entering a block: the norm before the projections, where latency is all
        {"name": "norm_fp8_decode", "op": "norm", "rows": 1, "k": 7168, "dtype": "bf16", "out": "fp8", "group": 128},
        # a ragged batch of prompts' tokens, one scale for each row
        {"name": "norm_fp8_ragged", "op": "norm", "rows": 777, "k": 4096, "dtype": "fp16", "out": "fp8", "group": 0},
        # a long prompt's tokens: memory traffic is all
        {"name": "norm_fp8_prompt", "op": "norm", "rows": 8192, "k": 7168, "dtype": "bf16", "out": "fp8", "group": 128},
        # a prompt chunk quantised for the NVFP4 GEMMs that follow
        {"name": "norm_nvfp4_prompt", "op": "norm", "rows": 2048, "k": 4096, "dtype": "bf16", "out": "nvfp4", "group": 16},
        # one token, a narrow projection: the smallest product, launch and latency count
        {"name": "gemv_1_narrow", "op": "gemv", "m": 1, "n": 1001, "k": 1536, "dtype": "bf16", "out": "bf16"},
        # one token through the down projection of a gated block
        {"name": "gemv_1_down", "op": "gemv", "m": 1, "n": 4096, "k": 14336, "dtype": "fp16", "out": "fp16"},
        # a small batch of decoded tokens, the long-K projection, sums kept in 32 bits
        {"name": "gemv_16_long", "op": "gemv", "m": 16, "n": 7168, "k": 16384, "dtype": "bf16", "out": "fp32"},
        # one token through both gate projections
        {"name": "dual_1", "op": "dual", "m": 1, "n": 14336, "k": 4096, "dtype": "bf16", "out": "bf16"},
        # an odd batch, odd width
        {"name": "dual_5_odd", "op": "dual", "m": 5, "n": 4099, "k": 7168, "dtype": "fp16", "out": "fp16"},
        # one token's experts, both gate projections
        {"name": "moe_dual_1", "op": "moe_dual", "tokens": 1, "topk": 8, "experts": 64, "n": 2048, "k": 7168, "dtype": "bf16", "out": "fp16"},
        # a small batch's experts, the down projection (a row for each choice)
        {"name": "moe_down_8", "op": "moe", "tokens": 8, "topk": 8, "experts": 64, "n": 7168, "k": 2048, "dtype": "fp16", "out": "fp16"},
        # the same for one token: few experts, latency counts
        {"name": "moe_down_1", "op": "moe", "tokens": 1, "topk": 2, "experts": 8, "n": 4096, "k": 1536, "dtype": "bf16", "out": "fp16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("norm", "norm", "gemv", "gemv", "dual", "moe", "moe_dual"))
    dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
    if op == "norm":
        out = rng.choice(("fp8", "nvfp4"))
        k = 128 * _log(rng, 2, 128)
        rows = min(_log(rng, 1, 8192), 8192 * 7168 // k // SIZE[dtype] * 2)
        group = 16 if out == "nvfp4" else rng.choice((0, 32, 64, 128))
        return {"op": op, "rows": rows, "k": k, "dtype": dtype, "out": out, "group": group}
    out = rng.choice((dtype, dtype, "fp32", "fp16"))
    if op in ("gemv", "dual"):
        k = 64 * _log(rng, 2, 256)
        most = 7168 * 16384 // k // (2 if op == "dual" else 1)
        return {"op": op, "m": _log(rng, 1, 16), "n": min(_log(rng, 16, 16384), most), "k": k, "dtype": dtype, "out": out}
    tokens, topk, experts = _log(rng, 1, 16), rng.choice((1, 2, 4, 8)), rng.choice((8, 16, 32, 64, 128))
    k = 64 * _log(rng, 4, 112)
    most = 7168 * 2048 * 64 // max(experts, tokens * topk) // k // (2 if op == "moe_dual" else 1)
    return {"op": op, "tokens": tokens, "topk": topk, "experts": experts, "n": min(_log(rng, 64, 7168), most), "k": k, "dtype": dtype, "out": out}


def work(case):
    op, e = case["op"], SIZE[case["dtype"]]
    if op == "norm":
        n = case["rows"] * case["k"]
        scales = case["rows"] * (4 * (case["k"] // case["group"] if case["group"] else 1) if case["out"] == "fp8" else case["k"] // 16)
        return {"bytes": n * (3 * e + (1 if case["out"] == "fp8" else 0.5)) + case["k"] * e + scales, "flops": 6 * n}
    n, k, both = case["n"], case["k"], 2 if op in ("dual", "moe_dual") else 1
    weights = n * k * 9 / 16 * both
    if op in ("gemv", "dual"):
        m = case["m"]
        return {"bytes": weights + m * k * e + m * n * SIZE[case["out"]], "flops": 2 * m * n * k * both}
    t, topk, x = case["tokens"], case["topk"], case["experts"]
    chosen = x * (1 - (1 - topk / x) ** t)  # different experts that the tokens choose, on the average
    rows = t if op == "moe_dual" else t * topk
    return {"bytes": chosen * weights + rows * k * e + t * topk * (4 + n * SIZE[case["out"]]), "flops": 2 * t * topk * n * k * both}


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _weights(g, experts, n, k):
    """NVFP4 weights as quantised normal values have them: codes with a normal distribution's
    frequencies, scales within a factor of eight of one another."""
    share = (3, 4, 5, 4, 7, 5, 3, 1)  # magnitudes 0 .. 6, of 32
    half = [c for c, s in enumerate(share) for _ in range(s)]
    nib = half + [c | 8 for c in half]
    table = torch.tensor([lo | hi << 4 for hi in nib for lo in nib], dtype=torch.uint8, device="cuda")
    packed = torch.empty((experts, n, k // 2), dtype=torch.uint8, device="cuda")
    for w in packed:
        w.copy_(table[torch.randint(0, 4096, w.shape, generator=g, device="cuda", dtype=torch.int32)])
    atoms = torch.randint(0x0C, 0x25, (experts, -(-n // 128), k // 64, 32, 4, 4), generator=g, device="cuda", dtype=torch.uint8)
    return packed, atoms


def _package():
    """This repository's package on the path, as its documentation has it."""
    if "blackwell-nvfp4-kernels_b200" not in sys.path:
        sys.path.insert(0, "blackwell-nvfp4-kernels_b200")


def _handle(kind, packed, atoms):
    """The weights as a program keeps them: nvfp4_b200's objects, made once."""
    _package()
    from nvfp4_b200 import gemv, moe
    if kind == "moe":
        return moe.ExpertWeights(list(zip(packed, atoms)))
    return gemv.Weights(packed[0], atoms[0])


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    op, t = case["op"], TYPES[case["dtype"]]
    s = {"case": case}
    if op == "norm":
        rows, k = case["rows"], case["k"]
        s["x"] = torch.randn(rows, k, generator=g, device="cuda").to(t)
        s["residual"] = (4 * torch.randn(rows, k, generator=g, device="cuda")).to(t)
        s["weight"] = (1 + 0.2 * torch.randn(k, generator=g, device="cuda")).to(t)
        if case["out"] == "nvfp4":   # a byte's two codes as two fp16 values, to read the packed output with
            values = torch.tensor(E2M1 + tuple(-v for v in E2M1), dtype=torch.float16, device="cuda")
            s["pairs"] = torch.stack((values.repeat(16), values.repeat_interleave(16)), 1).view(torch.int32).reshape(-1)
        return s
    moe = op in ("moe", "moe_dual")
    n, k = case["n"], case["k"]
    rows = case["m"] if not moe else case["tokens"] * (case["topk"] if op == "moe" else 1)
    s["x"] = torch.randn(rows, k, generator=g, device="cuda").to(t)
    if moe:
        s["ids"] = torch.rand(case["tokens"], case["experts"], generator=g, device="cuda").topk(case["topk"], dim=1).indices.to(torch.int32)
    for name in ("w1", "w2") if op in ("dual", "moe_dual") else ("w1",):
        s[name] = _weights(g, case["experts"] if moe else 1, n, k)
        if own:
            s[name + "_kept"] = _handle("moe" if moe else "dense", *s[name])
    return s


# ---------------------------------------------------------------------------
# Plain forms
# ---------------------------------------------------------------------------
def _dequantised(packed, atoms):
    """[..., N, K/2] codes and [..., ceil(N/128), K/64, 32, 4, 4] scales -> fp32 [..., N, K]."""
    table = torch.tensor(E2M1 + tuple(-v for v in E2M1), device=packed.device)
    codes = torch.stack((packed & 15, packed >> 4), dim=-1)
    lead, n, k = packed.shape[:-2], packed.shape[-2], packed.shape[-1] * 2
    values = table[codes.to(torch.int32)].reshape(*lead, n, k // 16, 16)
    scales = atoms.view(torch.float8_e4m3fn).float()
    d = scales.dim()
    scales = scales.permute(*range(len(lead)), d - 5, d - 2, d - 3, d - 4, d - 1)   # row blocks, quarters, rows of 32; atoms, blocks
    scales = scales.reshape(*lead, -1, k // 16)[..., :n, :]
    return (values * scales.unsqueeze(-1)).reshape(*lead, n, k)


def _e2m1(q):
    """Nearest e2m1 value, ties to the even code, saturating at 6."""
    a = q.abs()
    m = torch.zeros_like(a)
    m = torch.where(a > 0.25, 0.5, m)
    m = torch.where(a >= 0.75, 1.0, m)
    m = torch.where(a > 1.25, 1.5, m)
    m = torch.where(a >= 1.75, 2.0, m)
    m = torch.where(a > 2.5, 3.0, m)
    m = torch.where(a >= 3.5, 4.0, m)
    m = torch.where(a > 5.0, 6.0, m)
    return torch.copysign(m, q)


def _plain_norm(s):
    c, t = s["case"], s["x"].dtype
    rows, k = s["x"].shape
    h = (s["x"].float() + s["residual"].float()).to(t)
    mean = (h.double() * h.double()).sum(1, keepdim=True) / k   # a sum whose last bits decide borders of the codes
    r = (1.0 / torch.sqrt(mean + EPS)).float()
    y = h.float() * r * s["weight"].float()
    if c["out"] == "fp8":
        group = c["group"] or k
        y = y.reshape(rows, k // group, group)
        scale = y.abs().amax(2, keepdim=True) / 448.0
        q = torch.where(scale == 0, 0.0, y / scale).clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
        return {"h": h, "q": q.reshape(rows, k), "scale": scale.reshape(rows, -1)}
    y = y.reshape(rows, k // 16, 16)
    sf = (y.abs().amax(2) / 6.0).clamp(max=448.0).to(torch.float8_e4m3fn)
    d = sf.float().unsqueeze(2)
    q = _e2m1(torch.where(d == 0, 0.0, y / d)).reshape(rows, k).half()
    padded = torch.zeros(-(-rows // 128) * 128, k // 16, device=q.device)
    padded[:rows] = sf.float()
    atoms = padded.reshape(-1, 4, 32, k // 64, 4).permute(0, 3, 2, 1, 4).contiguous().to(torch.float8_e4m3fn)
    return {"h": h, "q": q, "sf": sf, "atoms": atoms}


def _gate(g, u):
    return g / (1 + torch.exp(-g)) * u


def _plain_product(s):
    c = s["case"]
    x, out = s["x"].float(), TYPES[c["out"]]
    if c["op"] in ("gemv", "dual"):
        y = [x @ _dequantised(*s[w])[0].T for w in ("w1", "w2") if w in s]
    else:
        pairs = s["ids"].reshape(-1).long()
        if c["op"] == "moe_dual":
            x = x.repeat_interleave(c["topk"], 0)
        y = [(_dequantised(*(v[pairs] for v in s[w])) @ x.unsqueeze(2)).squeeze(2) for w in ("w1", "w2") if w in s]
    return (_gate(*y) if len(y) == 2 else y[0]).to(out)


def _own(s):
    from nvfp4_b200 import gemv, moe, norm
    c = s["case"]
    if c["op"] == "norm":
        if c["out"] == "fp8":
            (q, scale), h = norm.rms_norm_fp8(s["x"], s["weight"], s["residual"], eps=EPS, group=c["group"] or None)
            return {"h": h, "q": q, "scale": scale}
        (packed, sf, atoms), h = norm.rms_norm_nvfp4(s["x"], s["weight"], s["residual"], eps=EPS)
        q = s["pairs"][packed.view(torch.uint8).reshape(-1).to(torch.int32)].view(torch.float16).reshape(c["rows"], c["k"])
        return {"h": h, "q": q, "sf": sf.reshape(c["rows"], -1), "atoms": atoms.permute(5, 2, 4, 0, 1, 3)[0]}
    out = TYPES[c["out"]]
    if c["op"] == "gemv":
        return gemv.gemv(s["x"], s["w1_kept"], out_dtype=out)
    if c["op"] == "dual":
        return gemv.dual_gemv(s["x"], s["w1_kept"], s["w2_kept"], out_dtype=out)
    if c["op"] == "moe":
        return moe.gemv(s["x"], s["ids"], s["w1_kept"], out_dtype=out)
    return moe.dual_gemv(s["x"], s["ids"], s["w1_kept"], s["w2_kept"], out_dtype=out)


def run(state):
    if own:
        _package()
        return _own(state)
    return _plain_norm(state) if state["case"]["op"] == "norm" else _plain_product(state)


# ---------------------------------------------------------------------------
# The definitions in 64 bits
# ---------------------------------------------------------------------------
def _decoded(packed, atoms):
    """One matrix in 64 bits from the formats' bit fields, scales found by their byte's address."""
    n, k = packed.shape[0], packed.shape[1] * 2
    code = torch.empty((n, k), dtype=torch.int64, device=packed.device)
    code[:, 0::2], code[:, 1::2] = packed.long() % 16, packed.long() // 16
    exp, man = code // 2 % 4, (code % 2).double()
    value = torch.where(exp == 0, man / 2, (1 + man / 2) * 2.0 ** (exp - 1).double())
    value = torch.where(code >= 8, -value, value)
    r = torch.arange(n, device=packed.device).unsqueeze(1)
    b = torch.arange(k // 16, device=packed.device).unsqueeze(0)
    at = ((r // 128) * (k // 64) + b // 4) * 512 + (r % 32) * 16 + (r % 128 // 32) * 4 + b % 4
    byte = atoms.reshape(-1)[at].long()
    exp, man = byte // 8 % 16, (byte % 8).double()
    scale = torch.where(exp == 0, man / 8 * 2.0 ** -6, (1 + man / 8) * 2.0 ** (exp - 7).double())
    return value * scale.repeat_interleave(16, 1)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        h = (s["x"].double() + s["residual"].double()).to(s["x"].dtype)
        v = h.double()
        y = v * (v.square().mean(1, keepdim=True) + EPS).rsqrt() * s["weight"].double()
        rows, k = y.shape
        if case["out"] == "fp8":
            group = case["group"] or k
            top = y.view(rows, -1, group).abs().max(2).values / 448
            q = (y / top.repeat_interleave(group, 1)).nan_to_num(0.0)
            step = 2.0 ** (q.abs().clamp(min=2.0 ** -6).log2().floor() - 3)
            return {"h": v, "q": ((q / step).round() * step).clamp(-448, 448), "scale": top}
        top = (y.view(rows, -1, 16).abs().max(2).values / 6).clamp(max=448)
        step = 2.0 ** (top.clamp(min=2.0 ** -6).log2().floor() - 3)
        sf = (top / step).round() * step
        q = (y / sf.repeat_interleave(16, 1)).nan_to_num(0.0).clamp(-6, 6)
        step = 2.0 ** (q.abs().clamp(min=1.0).log2().floor() - 1)
        r = torch.arange(rows, device=y.device).unsqueeze(1)
        b = torch.arange(k // 16, device=y.device).unsqueeze(0)
        atoms = torch.zeros(-(-rows // 128), k // 64, 32, 4, 4, dtype=torch.float64, device=y.device)
        atoms[r // 128, b // 4, r % 32, r % 128 // 32, b % 4] = sf
        return {"h": v, "q": (q / step).round() * step, "sf": sf, "atoms": atoms}
    x = s["x"].double()
    if case["op"] in ("gemv", "dual"):
        y = [x @ _decoded(s[w][0][0], s[w][1][0]).T for w in ("w1", "w2") if w in s]
    else:
        ids, y = s["ids"].reshape(-1).tolist(), []
        for w in ("w1", "w2"):
            if w in s:
                rows = torch.empty(len(ids), case["n"], dtype=torch.float64, device=x.device)
                for e in sorted(set(ids)):
                    d = _decoded(s[w][0][e], s[w][1][e])
                    for p, i in enumerate(ids):
                        if i == e:
                            rows[p] = d @ x[p if case["op"] == "moe" else p // case["topk"]]
                y.append(rows)
    return y[0] if len(y) == 1 else y[0] * torch.sigmoid(y[0]) * y[1]
