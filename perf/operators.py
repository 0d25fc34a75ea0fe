"""Timed cases of the 4-bit block and its norms: quantisation to microscaled
4-bit floating point (MXFP4: E2M1 elements, one E8M0 scale for 32 of them),
products of such matrices, the chained MLP on them, and the norms before and
after a block fused with its gate and residual scale, forward and backward.

Where `own` is true, run() makes the framework's calls; where it is false it
computes the same from elementary torch operations in 32 bits.  Both take the
operands of prepare().  A packed matrix of R rows and K columns is Q, uint8
[R, Kp / 2] with Kp = K rounded up to a multiple of 256 (two elements a byte,
the first in the low four bits), and S, uint8 [ceil(K / 512), R, 4, 4]: the
scales of 512 columns of a row together, that of its block b (of 32 columns)
at [b % 4, b / 4].  Elements and scales behind column K are zero.
"""
from __future__ import annotations

import math

import torch

own = False


# ------------------------------------------------------------------ the cases
def listed() -> list[dict]:
    return [
        # one token through the up-projection of the benchmark's MLP: quantise its row, multiply with the kept weights
        {"name": "linear_token", "op": "linear", "M": 1, "K": 4096, "N": 11008},
        # a ragged batch, no size a multiple of anything
        {"name": "linear_ragged", "op": "linear", "M": 333, "K": 1000, "N": 777},
        # a product of kept operands at the size of the bf16 benchmark, fp32 results
        {"name": "gemm_8192", "op": "gemm", "M": 8192, "K": 8192, "N": 8192, "out": "f32"},
        # a prompt of 2048 tokens through the MLP of the benchmark
        {"name": "mlp_2048", "op": "mlp", "M": 2048, "K": 4096, "F": 11008, "N": 4096},
        # eight tokens through the same MLP: the serving step
        {"name": "mlp_8", "op": "mlp", "M": 8, "K": 4096, "F": 11008, "N": 4096},
        # quantisation of a large activation along its rows, and its values (fake quantisation)
        {"name": "quant_8192", "op": "quant", "R": 8192, "C": 8192, "dtype": "bf16", "axis": "rows"},
        # quantisation along both axes, as the products of a backward pass need it, odd sizes, fp32 input
        {"name": "quant_both_odd", "op": "quant", "R": 1023, "C": 2049, "dtype": "f32", "axis": "both"},
        # gradients of a 4-bit linear layer: every operand quantised along the axis that its product contracts
        {"name": "linear_grad", "op": "linear_grad", "M": 2048, "K": 4096, "N": 4096},
        # one token through the norms of a block
        {"name": "norm_token", "op": "norm", "rows": 1, "cols": 4096, "stream": "bf16", "gate": "none", "before": True,
         "after": True, "grad": False},
        # a prompt: a gate for each sequence, a residual stream in fp32
        {"name": "norm_8192", "op": "norm", "rows": 8192, "cols": 4096, "stream": "f32", "gate": "group",
         "before": True, "after": True, "grad": False},
        # a training step's gradient through both norms, one gate vector, an uneven number of tokens
        {"name": "norm_grad_4095", "op": "norm", "rows": 4095, "cols": 4096, "stream": "bf16", "gate": "one",
         "before": True, "after": True, "grad": True},
        # the same of a small odd model: few tokens, rows of an odd length, a gate for each sequence
        {"name": "norm_grad_odd", "op": "norm", "rows": 333, "cols": 1111, "stream": "f32", "gate": "group",
         "before": True, "after": True, "grad": True},
    ]


def _size(rng, lo: int, hi: int) -> int:
    """Spread over the logarithm of [lo, hi]; a third each multiples of 128, of 32, and as they fall."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi + 0.999)))
    unit = rng.choice((128, 32, 1))
    n = round(v / unit) * unit if v >= unit else int(v)
    return min(hi, max(lo, n))


def draw(rng) -> dict:
    op = rng.choice(("linear", "linear", "gemm", "mlp", "quant", "linear_grad", "norm", "norm"))
    if op in ("linear", "gemm", "linear_grad"):
        while True:
            M, K, N = _size(rng, 1, 8192), _size(rng, 32, 12288), _size(rng, 16, 12288)
            if M * K * N <= (8192**3 if op == "gemm" else 2**36):
                break
        case = {"op": op, "M": M, "K": K, "N": N}
        if op == "gemm":
            case["out"] = rng.choice(("f32", "bf16"))
        return case
    if op == "mlp":
        while True:
            M, K, F, N = _size(rng, 1, 2048), _size(rng, 256, 4096), _size(rng, 256, 11008), _size(rng, 256, 4096)
            if M * F * (K + N) <= 2048 * 11008 * 8192:
                return {"op": op, "M": M, "K": K, "F": F, "N": N}
    if op == "quant":
        while True:
            R, C = _size(rng, 1, 16384), _size(rng, 1, 16384)
            if 2**10 <= R * C <= 2**26:
                return {"op": op, "R": R, "C": C, "dtype": rng.choice(("f32", "bf16")),
                        "axis": rng.choice(("rows", "columns", "both"))}
    while True:
        rows, cols = _size(rng, 1, 16384), _size(rng, 33, 8192)
        if rows * cols <= 2**25:
            break
    before, after = rng.choice(((True, True), (True, True), (True, False), (False, True)))
    return {"op": "norm", "rows": rows, "cols": cols, "stream": rng.choice(("f32", "bf16")),
            "gate": rng.choice(("none", "one", "group", "row")) if after else "none", "before": before, "after": after,
            "grad": rng.random() < 0.5}


# ------------------------------------------------------------------ inputs
_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
_ALPHA, _EPS = 0.875, 1e-5  # residual scale, and the term under the norms' roots


def _padded(k: int, unit: int = 256) -> int:
    return (k + unit - 1) // unit * unit


def _gate_rows(c: dict) -> int:
    """Rows that share a row of the gate: all of them, a quarter (sequences of a batch), or each its own."""
    return {"none": c["rows"], "one": c["rows"], "group": -(-c["rows"] // 4), "row": 1}[c["gate"]]


def _empty(dtype, *shape):
    return torch.empty(shape, dtype=dtype, device="cuda")


def _inputs(case: dict, seed: int) -> dict:
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(*shape, scale=1.0):
        return torch.randn(shape, device="cuda", generator=g) * scale

    def activation(rows, cols, dtype=torch.bfloat16):
        """Normal values with a few columns some times as large, as hidden states have them."""
        return (normal(rows, cols) * torch.exp2(3 * torch.rand(cols, device="cuda", generator=g)**8)).to(dtype)

    def weight(rows, cols):
        """Packed weights as a program keeps them: N(0, 1 / cols), quantised once."""
        return _quantised(normal(rows, cols, scale=cols**-0.5))

    op = case["op"]
    if op == "linear":
        return {"X": activation(case["M"], case["K"]), "W": weight(case["N"], case["K"])}
    if op == "gemm":
        return {"A": _quantised(activation(case["M"], case["K"])), "B": weight(case["N"], case["K"])}
    if op == "mlp":
        return {"X": activation(case["M"], case["K"]), "W1": weight(case["F"], case["K"]),
                "W2": weight(case["N"], case["F"])}
    if op == "quant":
        return {"X": activation(case["R"], case["C"], _DTYPES[case["dtype"]])}
    if op == "linear_grad":
        return {"dY": normal(case["M"], case["N"], scale=1e-3).to(torch.bfloat16),
                "X": activation(case["M"], case["K"]),
                "W": normal(case["N"], case["K"], scale=case["K"]**-0.5).to(torch.bfloat16)}
    rows, cols, stream = case["rows"], case["cols"], _DTYPES[case["stream"]]
    s = {"x": activation(rows, cols, stream)}
    if case["after"]:
        s["b"] = normal(rows, cols, scale=0.5).to(torch.bfloat16)
        s["w_after"] = 1 + normal(cols, scale=0.1)
        if case["gate"] != "none":
            s["gate"] = (1 + normal(-(-rows // _gate_rows(case)), cols, scale=0.3)).to(torch.bfloat16)
    if case["before"]:
        s["w_before"] = 1 + normal(cols, scale=0.1)
    if case["grad"]:
        # what the forward pass leaves, and the gradients that arrive
        f = _norm_forward(case, s)
        s["out"], s["rstd"] = f["out"], f["rstd"]
        s["dout"] = normal(rows, cols, scale=1e-2).to(stream)
        if case["before"]:
            s["dy"] = normal(rows, cols, scale=1e-2).to(torch.bfloat16)
    return s


def prepare(case: dict, seed: int) -> dict:
    """The inputs, and the buffers that a program keeps for the packed operands and the results."""
    s = _inputs(case, seed)
    op, u8, bf, f32 = case["op"], torch.uint8, torch.bfloat16, torch.float32

    def packed(rows, cols):
        return _empty(u8, rows, _padded(cols) // 2), _empty(u8, _padded(cols, 512) // 512, rows, 4, 4)

    if op == "linear":
        s["Xq"], s["Y"] = packed(case["M"], case["K"]), _empty(bf, case["M"], case["N"])
    elif op == "gemm":
        s["C"] = _empty(_DTYPES[case["out"]], case["M"], case["N"])
    elif op == "mlp":
        s["Xq"], s["Hq"], s["Y"] = packed(case["M"], case["K"]), packed(case["M"], case["F"]), _empty(bf, case["M"], case["N"])
    elif op == "quant":
        R, C = case["R"], case["C"]
        if case["axis"] != "columns":
            s["Xq"], s["V"] = packed(R, C), _empty(bf, R, C)
        if case["axis"] != "rows":
            s["Xt"], s["Vt"] = packed(C, R), _empty(bf, C, R)
    elif op == "linear_grad":
        M, N, K = case["M"], case["N"], case["K"]
        s["dYq"], s["dYt"], s["Xt"], s["Wt"] = packed(M, N), packed(N, M), packed(K, M), packed(K, N)
        s["dX"], s["dW"] = _empty(bf, M, K), _empty(f32, N, K)
    else:
        rows, cols, stream = case["rows"], case["cols"], _DTYPES[case["stream"]]
        if not case["grad"]:
            s["rstd_"] = _empty(f32, 2, rows)
            if case["after"]:
                s["out_"] = _empty(stream, rows, cols)
            if case["before"]:
                s["y_"] = _empty(bf, rows, cols)
        else:
            s["work"] = _empty(f32, 1024 * cols)
            s["dx_"] = _empty(stream, rows, cols)
            if case["after"]:
                s["db_"], s["dw_after_"] = _empty(bf, rows, cols), _empty(f32, cols)
                if case["gate"] != "none":
                    s["dgate_"] = _empty(f32, *s["gate"].shape)
            if case["before"]:
                s["dw_before_"] = _empty(f32, cols)
    s["case"] = dict(case)
    return s


# ------------------------------------------------------------------ one pass
def run(state: dict):
    return _run_own(state) if own else _run_plain(state)


# ------------------------------------------------------------------ ... through the framework
_contexts: dict = {}


def _context():
    """The program's one context per stream."""
    stream = torch.cuda.current_stream().cuda_stream
    if stream not in _contexts:
        import aiehlc_amd as mi

        _contexts[stream] = mi.Context(torch.cuda.current_device(), stream=stream)
    return _contexts[stream]


_F32, _BF16 = 0, 1  # the framework's names of the element types
_CODE = {torch.float32: _F32, torch.bfloat16: _BF16}


def _p(t):
    return None if t is None else t.data_ptr()


def _pp(pair):
    return pair[0].data_ptr(), pair[1].data_ptr()


def _run_own(s: dict):
    c, ctx = s["case"], _context()
    op = c["op"]
    if op == "linear":
        M, K, N = c["M"], c["K"], c["N"]
        xq, wq = _pp(s["Xq"]), _pp(s["W"])
        ctx.quant_mxfp4(_p(s["X"]), M, K, *xq, dtype=_BF16)
        ctx.gemm_mxfp4(*xq, *wq, _p(s["Y"]), M, N, K, dtype=_BF16)
        return s["Y"]
    if op == "gemm":
        ctx.gemm_mxfp4(*_pp(s["A"]), *_pp(s["B"]), _p(s["C"]), c["M"], c["N"], c["K"], dtype=_CODE[s["C"].dtype])
        return s["C"]
    if op == "mlp":
        M, K, F, N = c["M"], c["K"], c["F"], c["N"]
        xq = _pp(s["Xq"])
        ctx.quant_mxfp4(_p(s["X"]), M, K, *xq, dtype=_BF16)
        ctx.mlp_mxfp4(*xq, *_pp(s["W1"]), *_pp(s["W2"]), *_pp(s["Hq"]), _p(s["Y"]), M, K, F, N, dtype=_BF16)
        return s["Y"]
    if op == "quant":
        R, C, X = c["R"], c["C"], s["X"]
        q, qt = s.get("Xq"), s.get("Xt")
        ctx.quant_mxfp4(_p(X), R, C, *(_pp(q) if q else (None, None)), *(_pp(qt) if qt else (None, None)),
                        dtype=_CODE[X.dtype])
        out = []
        if q:
            ctx.dequant_mxfp4(*_pp(q), _p(s["V"]), R, C, dtype=_BF16)
            out.append(s["V"])
        if qt:
            ctx.dequant_mxfp4(*_pp(qt), _p(s["Vt"]), C, R, dtype=_BF16)
            out.append(s["Vt"])
        return out
    if op == "linear_grad":
        M, N, K = c["M"], c["N"], c["K"]
        dyq, dyt, xt, wt = (_pp(s[k]) for k in ("dYq", "dYt", "Xt", "Wt"))
        ctx.quant_mxfp4(_p(s["dY"]), M, N, *dyq, *dyt, dtype=_BF16)
        ctx.quant_mxfp4(_p(s["X"]), M, K, None, None, *xt, dtype=_BF16)
        ctx.quant_mxfp4(_p(s["W"]), N, K, None, None, *wt, dtype=_BF16)
        ctx.gemm_mxfp4(*dyq, *wt, _p(s["dX"]), M, K, N, dtype=_BF16)
        ctx.gemm_mxfp4(*dyt, *xt, _p(s["dW"]), N, K, M, dtype=_F32)
        return s["dX"], s["dW"]
    rows, cols, stream = c["rows"], c["cols"], _CODE[s["x"].dtype]
    if not c["grad"]:
        ctx.norm_block(_p(s["x"]), _p(s.get("b")), _p(s.get("gate")), _p(s.get("w_after")), _p(s.get("w_before")),
                       _p(s.get("out_")), _p(s.get("y_")), _p(s["rstd_"]), rows, cols, gate_rows=_gate_rows(c),
                       stream_dtype=stream, branch_dtype=_BF16, alpha=_ALPHA, eps=_EPS)
        return {k: s[k + "_"] for k in ("out", "y") if k + "_" in s}
    ctx.norm_block_grad(_p(s["out"]), _p(s.get("b")), _p(s.get("gate")), _p(s.get("w_after")), _p(s.get("w_before")),
                        _p(s["rstd"]), _p(s["dout"]), _p(s.get("dy")), _p(s["dx_"]), _p(s.get("db_")),
                        _p(s.get("dgate_")), _p(s.get("dw_after_")), _p(s.get("dw_before_")), _p(s["work"]),
                        4 * s["work"].numel(), rows, cols, gate_rows=_gate_rows(c), stream_dtype=stream,
                        branch_dtype=_BF16, alpha=_ALPHA)
    return {k: s[k + "_"] for k in ("dx", "db", "dgate", "dw_after", "dw_before") if k + "_" in s}


# ------------------------------------------------------------------ ... in plain form
def _e2m1(device):
    return torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], device=device)


def _quantised(X: torch.Tensor):
    """(Q, S) of a matrix, along its rows."""
    R, K = X.shape
    x = torch.nn.functional.pad(X.float(), (0, _padded(K, 512) - K)).reshape(R, -1, 32)
    amax = x.abs().amax(-1)
    # 2^e scales the block so that its largest value falls into [4, 8); E2M1 ends at 6
    e = torch.where(amax > 0, torch.frexp(amax).exponent - 3, -127).clamp(min=-127)
    y = x * torch.exp2(-e.float()).unsqueeze(-1)
    a = y.abs()
    # E2M1 steps by 0.5 below 2, by 1 below 4, by 2 below 8; codes 0-3, 4-5, 6-7 (halves to the even code)
    code = torch.where(a < 2, torch.round(a * 2), torch.where(a < 4, torch.round(a) + 2, torch.round(a * 0.5) + 4))
    code = code.clamp(max=7).to(torch.uint8) | ((y < 0) * 8).to(torch.uint8)
    code = code.reshape(R, -1, 2)[:, :_padded(K) // 2]
    S = (e + 127).to(torch.uint8).reshape(R, -1, 4, 4).permute(1, 0, 3, 2)
    return code[..., 0] | (code[..., 1] << 4), S.contiguous()


def _values(Q: torch.Tensor, S: torch.Tensor, K: int) -> torch.Tensor:
    """The fp32 values that a packed matrix stands for."""
    R = Q.shape[0]
    code = torch.stack((Q & 15, Q >> 4), -1).reshape(R, -1, 32)
    scale = torch.exp2(S.float() - 127).permute(1, 0, 3, 2).reshape(R, -1)[:, :code.shape[1]]
    return (_e2m1(Q.device)[code.int()] * scale.unsqueeze(-1)).reshape(R, -1)[:, :K]


def _rounded(X: torch.Tensor) -> torch.Tensor:
    """X rounded to MXFP4 along its rows."""
    return _values(*_quantised(X), X.shape[1])


def _columns(X: torch.Tensor) -> torch.Tensor:
    return X.t().contiguous()


def _norm_forward(c: dict, s: dict) -> dict:
    cols, r = c["cols"], s["x"].float()
    rstd = torch.zeros(2, c["rows"], device=r.device)
    got = {"out": s["x"], "rstd": rstd}
    if c["after"]:
        b = s["b"].float()
        rstd[0] = torch.rsqrt(b.square().mean(-1) + _EPS)
        n = b * rstd[0].unsqueeze(-1) * s["w_after"]
        if "gate" in s:
            n = n * s["gate"].float().repeat_interleave(_gate_rows(c), 0)[:c["rows"]]
        got["out"] = (_ALPHA * r + n).to(s["x"].dtype)
        r = got["out"].float()
    if c["before"]:
        rstd[1] = torch.rsqrt(r.square().mean(-1) + _EPS)
        got["y"] = (r * rstd[1].unsqueeze(-1) * s["w_before"]).to(torch.bfloat16)
    return got


def _norm_backward(c: dict, s: dict) -> dict:
    got, dr = {}, s["dout"].float()
    ra, rb = s["rstd"][0].unsqueeze(-1), s["rstd"][1].unsqueeze(-1)
    if c["before"]:
        m, dy = s["out"].float() * rb, s["dy"].float()
        t = dy * s["w_before"]
        got["dw_before"] = (dy * m).sum(0)
        dr = dr + rb * (t - m * (t * m).mean(-1, keepdim=True))
    got["dx"] = ((_ALPHA if c["after"] else 1.0) * dr).to(s["dout"].dtype)
    if c["after"]:
        n, d = s["b"].float() * ra, dr
        if "gate" in s:
            k, G = _gate_rows(c), s["gate"].shape[0]
            p = torch.nn.functional.pad(dr * n * s["w_after"], (0, 0, 0, G * k - c["rows"]))
            got["dgate"] = p.reshape(G, k, -1).sum(1)
            d = dr * s["gate"].float().repeat_interleave(k, 0)[:c["rows"]]
        got["dw_after"] = (d * n).sum(0)
        u = d * s["w_after"]
        got["db"] = (ra * (u - n * (u * n).mean(-1, keepdim=True))).to(torch.bfloat16)
    return got


def _run_plain(s: dict):
    c = s["case"]
    op = c["op"]
    if op == "linear":
        return (_rounded(s["X"]) @ _values(*s["W"], c["K"]).t()).to(torch.bfloat16)
    if op == "gemm":
        return (_values(*s["A"], c["K"]) @ _values(*s["B"], c["K"]).t()).to(_DTYPES[c["out"]])
    if op == "mlp":
        H = (_rounded(s["X"]) @ _values(*s["W1"], c["K"]).t()).clamp_(min=0)
        return (_rounded(H) @ _values(*s["W2"], c["F"]).t()).to(torch.bfloat16)
    if op == "quant":
        out = []
        if c["axis"] != "columns":
            out.append(_rounded(s["X"]).to(torch.bfloat16))
        if c["axis"] != "rows":
            out.append(_rounded(_columns(s["X"])).to(torch.bfloat16))
        return out
    if op == "linear_grad":
        dX = _rounded(s["dY"]) @ _rounded(_columns(s["W"])).t()
        dW = _rounded(_columns(s["dY"])) @ _rounded(_columns(s["X"])).t()
        return dX.to(torch.bfloat16), dW
    if c["grad"]:
        got = _norm_backward(c, s)
        return {k: got[k] for k in ("dx", "db", "dgate", "dw_after", "dw_before") if k in got}
    got = _norm_forward(c, s)
    return {k: got[k] for k in (("out",) if c["after"] else ()) + (("y",) if c["before"] else ())}


# ------------------------------------------------------------------ what a pass cannot do without
def work(case: dict) -> dict:
    def fp4(rows, cols):
        return rows * cols * 17 / 32

    op = case["op"]
    if op in ("linear", "gemm"):
        M, N, K = case["M"], case["N"], case["K"]
        inb = 2 * M * K if op == "linear" else fp4(M, K)
        outb = (4 if case.get("out") == "f32" else 2) * M * N
        return {"bytes": inb + fp4(N, K) + outb, "flops": 2 * M * N * K}
    if op == "mlp":
        M, K, F, N = case["M"], case["K"], case["F"], case["N"]
        return {"bytes": 2 * M * K + fp4(F, K) + fp4(N, F) + 2 * M * N, "flops": 2 * M * F * (K + N)}
    if op == "quant":  # the packed matrices, written once, and the values
        n, k = case["R"] * case["C"], 2 if case["axis"] == "both" else 1
        return {"bytes": (2 if case["dtype"] == "bf16" else 4) * n + k * (17 / 32 + 2) * n, "flops": 0}
    if op == "linear_grad":
        M, N, K = case["M"], case["N"], case["K"]
        return {"bytes": 2 * (M * N + M * K + N * K) + 2 * M * K + 4 * N * K, "flops": 4 * M * N * K}
    n, st = case["rows"] * case["cols"], 2 if case["stream"] == "bf16" else 4
    gate = 0 if case["gate"] == "none" else 2 * -(-case["rows"] // _gate_rows(case)) * case["cols"]
    if not case["grad"]:
        b = st * n + (2 * n + gate + st * n if case["after"] else 0) + (2 * n if case["before"] else 0)
    else:
        b = 2 * st * n + (4 * n + 3 * gate if case["after"] else 0) + ((st + 2) * n if case["before"] else 0)
    return {"bytes": b, "flops": 0}


# ------------------------------------------------------------------ the same in 64 bits
def _exact_values(Q, S, K):
    """Values of a packed matrix from the fields of its codes: sign, two exponent bits, one mantissa bit."""
    out = torch.empty(Q.shape[0], 2 * Q.shape[1], dtype=torch.float64, device=Q.device)
    for half, code in ((0, Q & 15), (1, Q >> 4)):
        exponent, mantissa = ((code >> 1) & 3).double(), (code & 1).double()
        size = torch.where(exponent > 0, (1 + mantissa / 2) * torch.exp2(exponent - 1), mantissa / 2)
        out[:, half::2] = torch.where(code >= 8, -size, size)
    block = torch.arange(K, device=Q.device) // 32  # of each column
    scale = S[block // 16, :, block % 4, block % 16 // 4].t()
    return out[:, :K] * torch.exp2(scale.double() - 127)


def _exact_rounded(X):
    """The nearest E2M1 multiple of each block's power of two, found between the midpoints of neighbours."""
    R, K = X.shape
    x = torch.nn.functional.pad(X.double(), (0, -K % 32)).reshape(R, -1, 32)
    amax = x.abs().amax(-1, keepdim=True)
    scale = torch.exp2((torch.floor(torch.log2(amax.clamp(min=2.0**-140))) - 2).clamp(min=-127))
    a = x.abs() / scale
    grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=X.device)
    size = torch.zeros_like(a)
    for i in range(7):
        mid = (grid[i] + grid[i + 1]) / 2
        up = a >= mid if i % 2 else a > mid  # a value halfway goes to the neighbour with the even code
        size = torch.where(up, grid[i + 1], size)
    return (torch.sign(x) * size * scale).reshape(R, -1)[:, :K]


def _exact_product(A, B):
    return A.contiguous() @ B.t().contiguous()


def exact(case: dict, seed: int):
    s, op = _inputs(case, seed), case["op"]
    if op == "linear":
        return _exact_product(_exact_rounded(s["X"]), _exact_values(*s["W"], case["K"]))
    if op == "gemm":
        return _exact_product(_exact_values(*s["A"], case["K"]), _exact_values(*s["B"], case["K"]))
    if op == "mlp":
        H = _exact_product(_exact_rounded(s["X"]), _exact_values(*s["W1"], case["K"]))
        return _exact_product(_exact_rounded(torch.relu(H)), _exact_values(*s["W2"], case["F"]))
    if op == "quant":
        X = s["X"].double()
        return [_exact_rounded(m) for m, a in ((X, "columns"), (X.t(), "rows")) if case["axis"] != a]
    if op == "linear_grad":
        dY, X, W = s["dY"].double(), s["X"].double(), s["W"].double()
        return (_exact_product(_exact_rounded(dY), _exact_rounded(W.t())),
                _exact_product(_exact_rounded(dY.t()), _exact_rounded(X.t())))
    return _exact_norm_grad(case, s) if case["grad"] else _exact_norm(case, s)


def _exact_gate(case, s):
    if "gate" not in s:
        return torch.ones(1, 1, dtype=torch.float64, device="cuda")
    row = torch.arange(case["rows"], device="cuda") // _gate_rows(case)
    return s["gate"].double()[row]


def _exact_norm(case, s):
    """(the second norm reads the residual stream as it is stored)"""
    r, got = s["x"].double(), {}
    if case["after"]:
        b = s["b"].double()
        r = _ALPHA * r + _exact_gate(case, s) * s["w_after"].double() * b / torch.sqrt((b * b).mean(1, keepdim=True) + _EPS)
        got["out"] = r
        r = r.to(s["x"].dtype).double()
    if case["before"]:
        got["y"] = s["w_before"].double() * r / torch.sqrt((r * r).mean(1, keepdim=True) + _EPS)
    return got


def _exact_norm_grad(case, s):
    """Gradients by torch's own differentiation of the forward formulas in 64 bits, at the stored residual stream."""
    got, dr = {}, s["dout"].double()
    if case["before"]:
        r = s["out"].double().requires_grad_()
        w = s["w_before"].double().requires_grad_()
        y = w * r / torch.sqrt((r * r).mean(1, keepdim=True) + _EPS)
        d, got["dw_before"] = torch.autograd.grad(y, (r, w), s["dy"].double())
        dr = dr + d
    got["dx"] = dr * (_ALPHA if case["after"] else 1.0)
    if case["after"]:
        b, w = s["b"].double().requires_grad_(), s["w_after"].double().requires_grad_()
        g = s["gate"].double().requires_grad_() if "gate" in s else None
        n = w * b / torch.sqrt((b * b).mean(1, keepdim=True) + _EPS)
        if g is not None:
            n = n * g[torch.arange(case["rows"], device="cuda") // _gate_rows(case)]
        grads = torch.autograd.grad(n, (b, w) + ((g,) if g is not None else ()), dr)
        got["db"], got["dw_after"] = grads[:2]
        if g is not None:
            got["dgate"] = grads[2]
    return {k: got[k] for k in ("dx", "db", "dgate", "dw_after", "dw_before") if k in got}
