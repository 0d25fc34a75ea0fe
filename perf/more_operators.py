"""Timed cases of the 8-bit floating point products with a scale for each block
of 128, of the routing of tokens to experts, and of the experts' products: their
MLP from the routing to the weighted sum, forward and backward.

Where `own` is true, run() makes the framework's calls; where it is false it
computes the same from elementary torch operations.  Both take the operands of
prepare().

A packed matrix of R rows and K columns is Q, uint8 [R, Kp] with Kp = K rounded
up to a multiple of 128 (E4M3 elements, zero behind column K), and S, fp32
[Kp / 128, ceil(R / block)]: the scale of 128 columns of `block` rows (1, or 128
for weights).  Quantisation takes the smallest power of two that the block's
largest magnitude is at most 448 times, at least 2^-126; kept weights may have
any scale.

Slots: the rows (token, choice) sorted by expert, each expert's from a multiple
of 128 on, in the order of their tokens.
"""
from __future__ import annotations

import math

import torch

own = False


# ------------------------------------------------------------------ the cases
def listed() -> list[dict]:
    # an MLP of 64 experts, eight of them for a token, chosen by sigmoid scores with a bias for balance
    mlp = {"op": "experts", "E": 64, "k": 8, "D": 4096, "F": 1024, "scoring": "sigmoid", "bias": True, "masked": False}
    return [
        # one token through the up-projection of the benchmark's MLP: quantise its row, multiply with the kept weights
        {"name": "linear_token", "op": "linear", "M": 1, "K": 4096, "N": 11008},
        # a ragged batch, no size a multiple of anything
        {"name": "linear_ragged", "op": "linear", "M": 333, "K": 1000, "N": 777},
        # a product of kept operands at the size of the bf16 benchmark
        {"name": "gemm_8192", "op": "gemm", "M": 8192, "K": 8192, "N": 8192},
        # gradients of a linear layer: operands quantised along the axis that each product contracts
        {"name": "linear_grad", "op": "linear_grad", "M": 2048, "K": 4096, "N": 4096},
        # quantisation of the benchmark's up-projection weights in blocks of 128 x 128, and their transpose
        {"name": "quant_weights", "op": "quant", "R": 11008, "C": 4096, "dtype": "bf16", "block": 128, "axis": "both"},
        # routing of a serving step's tokens: sigmoid scores, a bias for balance, four of eight groups, eight experts
        {"name": "route_8", "op": "route", "T": 8, "E": 256, "k": 8, "scoring": "sigmoid", "bias": True, "groups": 8,
         "kept": 4, "grad": False, "masked": False},
        # routing of a long prompt: softmax scores, four experts
        {"name": "route_8192", "op": "route", "T": 8192, "E": 128, "k": 4, "scoring": "softmax", "bias": False,
         "groups": 1, "kept": 1, "grad": False, "masked": False},
        # the gradient of the weights with respect to the logits, an uneven number of tokens, some of them padding
        {"name": "route_grad_4095", "op": "route", "T": 4095, "E": 64, "k": 6, "scoring": "softmax", "bias": False,
         "groups": 1, "kept": 1, "grad": True, "masked": True},
        # the serving step of a batch of eight: nearly every token has experts of its own
        {"name": "experts_8", **mlp, "T": 8},
        # a prompt through the same experts
        {"name": "experts_2048", **mlp, "T": 2048},
        # a ragged model and a padded batch
        {"name": "experts_ragged", "op": "experts", "T": 333, "E": 7, "k": 2, "D": 1000, "F": 384, "scoring": "softmax",
         "bias": False, "masked": True},
        # a training step's gradients: of the tokens, both weights of every expert, and the logits
        {"name": "experts_grad", "op": "experts_grad", "T": 1023, "E": 8, "k": 2, "D": 2048, "F": 1024,
         "scoring": "softmax", "bias": False, "masked": False},
    ]


def _size(rng, lo: int, hi: int) -> int:
    """Spread over the logarithm of [lo, hi]; a third each multiples of 128, of 32, and as they fall."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi + 0.999)))
    unit = rng.choice((128, 32, 1))
    n = round(v / unit) * unit if v >= unit else int(v)
    return min(hi, max(lo, n))


def draw(rng) -> dict:
    op = rng.choice(("linear", "linear", "gemm", "quant", "linear_grad", "route", "route", "experts", "experts",
                     "experts_grad"))
    if op in ("linear", "gemm", "linear_grad"):
        while True:
            M, K, N = _size(rng, 1, 8192), _size(rng, 32, 12288), _size(rng, 16, 12288)
            if M * K * N <= (8192**3 if op == "gemm" else 2**36):
                break
        return {"op": op, "M": M, "K": K, "N": N}
    if op == "quant":
        while True:
            R, C = _size(rng, 1, 16384), _size(rng, 1, 16384)
            if 2**10 <= R * C <= 2**25:
                return {"op": op, "R": R, "C": C, "dtype": rng.choice(("f32", "bf16")), "block": rng.choice((1, 128)),
                        "axis": rng.choice(("rows", "columns", "both"))}
    scoring, bias, masked = rng.choice(("softmax", "sigmoid")), rng.random() < 0.5, rng.random() < 0.3
    if op == "route":
        grad = rng.random() < 0.4
        groups = rng.choice((1, 1, 4, 8))
        E = groups * _size(rng, 2, 512 // groups)
        kept = 1 if groups == 1 else rng.randint(1, groups)
        k = min(rng.randint(2 if grad else 1, 8), kept * (E // groups))  # (a single renormalised weight has no gradient)
        return {"op": op, "T": _size(rng, 1, 8192), "E": E, "k": k, "scoring": scoring, "bias": bias, "groups": groups,
                "kept": kept, "grad": grad, "masked": masked}
    most_work, most_weights = (2**36, 2**28) if op == "experts" else (2**32, 2**25)
    while True:
        T, E, D = _size(rng, 1, 4096), rng.randint(2, 128), _size(rng, 64, 4096)
        F, k = 128 * rng.randint(1, 16), rng.randint(2 if op == "experts_grad" else 1, 8)
        if k <= E and E * D * F <= most_weights and T * k * D * F <= most_work and E * T * D * F <= 2**39:
            return {"op": op, "T": T, "E": E, "k": k, "D": D, "F": F, "scoring": scoring, "bias": bias, "masked": masked}


# ------------------------------------------------------------------ inputs
_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
_SCALE = 2.5  # of the chosen experts' weights
_NONE = float("-inf")  # the logit of an expert that is not to be chosen


def _up(n: int, unit: int = 128) -> int:
    return -(-n // unit) * unit


def _slots(c: dict) -> int:
    """Rows that hold the slots of any routing of T tokens to k of E experts."""
    n = c["T"] * c["k"]
    used = min(c["E"], n)
    return 128 * (used + (n - used) // 128)


def _empty(dtype, *shape):
    return torch.empty(shape, dtype=dtype, device="cuda")


class _Random:
    def __init__(self, seed: int):
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed(seed)

    def normal(self, *shape, scale=1.0):
        return torch.randn(shape, device="cuda", generator=self.g) * scale

    def activation(self, rows, cols, dtype=torch.bfloat16):
        """Normal values with a few columns some times as large, as hidden states have them."""
        return (self.normal(rows, cols) * torch.exp2(3 * torch.rand(cols, device="cuda", generator=self.g)**8)).to(dtype)

    def weight(self, rows, cols):
        """Weights N(0, 1 / cols) as a program loads them: blocks of 128 x 128, scales that no power of two is near."""
        return _quantised(self.normal(rows, cols, scale=cols**-0.5), 128, lambda amax: amax / 448)

    def weights(self, experts, rows, cols):
        packed = [self.weight(rows, cols) for _ in range(experts)]
        return torch.stack([p[0] for p in packed]), torch.stack([p[1] for p in packed])

    def logits(self, c):
        """Some experts are liked better than others; the last tenth of a masked batch is padding."""
        x = self.normal(c["T"], c["E"]) + self.normal(c["E"], scale=0.5)
        if c["masked"]:
            x[c["T"] - c["T"] // 10:] = _NONE
        return x


def _inputs(c: dict, seed: int) -> dict:
    r, op, bf = _Random(seed), c["op"], torch.bfloat16
    if op == "linear":
        return {"X": r.activation(c["M"], c["K"]), "W": r.weight(c["N"], c["K"])}
    if op == "gemm":
        return {"A": _quantised(r.activation(c["M"], c["K"]), 1), "B": r.weight(c["N"], c["K"])}
    if op == "linear_grad":
        W = r.weight(c["N"], c["K"])
        return {"dY": r.normal(c["M"], c["N"], scale=1e-3).to(bf), "X": r.activation(c["M"], c["K"]),
                "Wt": _transposed(W, c["N"], c["K"])}
    if op == "quant":
        return {"X": r.activation(c["R"], c["C"], _DTYPES[c["dtype"]])}
    s = {"logits": r.logits(c)}
    if c["bias"]:
        s["bias"] = r.normal(c["E"], scale=0.05)
    if op == "route":
        if c["grad"]:
            s["idx"], s["w"] = _route(c, s)
            s["dw"] = r.normal(c["T"], c["k"], scale=1e-2)
        return s
    T, E, D, F = c["T"], c["E"], c["D"], c["F"]
    s["X"] = r.activation(T, D)
    W1, W2 = r.weights(E, 2 * F, D), r.weights(E, D, F)
    if op == "experts":
        s["W1"], s["W2"] = W1, W2
        return s
    # a training step: the packed transposes that the gradients contract along, and what the forward pass left
    s["W1t"], s["W2t"] = _transposed(W1, 2 * F, D), _transposed(W2, D, F)
    s["idx"], s["w"] = _route(c, s)
    s["dout"] = r.normal(T, D, scale=1e-2).to(bf)
    _slot_tables(c, s)
    R = _slots(c)
    s["GU"], s["Y"] = torch.zeros(R, 2 * F, dtype=bf, device="cuda"), torch.zeros(R, D, dtype=bf, device="cuda")
    X = _rounded(s["X"])
    for e in range(E):
        rows = s["row"][e][:int(s["count"][e])]
        if len(rows) == 0:
            continue
        at = slice(int(s["start"][e]), int(s["start"][e]) + len(rows))
        s["GU"][at] = (X[rows] @ _values(W1[0][e], W1[1][e], 2 * F, D).t()).to(bf)
        s["Y"][at] = (_rounded(_swiglu(s["GU"][at])) @ _values(W2[0][e], W2[1][e], D, F).t()).to(bf)
    return s


def _slot_tables(c: dict, s: dict) -> None:
    """count[e] tokens of expert e, start[e] its first slot, row[e] its tokens in order (then the others)."""
    hit = (s["idx"].unsqueeze(-1) == torch.arange(c["E"], device="cuda")).any(1)  # [T][E]
    s["count"] = hit.sum(0)
    s["start"] = torch.cumsum((s["count"] + 127) // 128 * 128, 0) - (s["count"] + 127) // 128 * 128
    s["row"] = torch.argsort((~hit).int(), dim=0, stable=True).t().contiguous()


def prepare(case: dict, seed: int) -> dict:
    """The inputs, and the buffers that a program keeps for the packed operands, the slots and the results."""
    c, s = case, _inputs(case, seed)
    op, u8, bf, f32, i32 = case["op"], torch.uint8, torch.bfloat16, torch.float32, torch.int32

    def packed(rows, cols, block=1):
        return _empty(u8, rows, _up(cols)), _empty(f32, _up(cols) // 128, -(-rows // block))

    if op == "linear":
        s["Xq"], s["C"] = packed(c["M"], c["K"]), _empty(bf, c["M"], c["N"])
    elif op == "gemm":
        s["C"] = _empty(bf, c["M"], c["N"])
    elif op == "linear_grad":
        M, N, K = c["M"], c["N"], c["K"]
        s["dYq"], s["dYt"], s["Xt"] = packed(M, N), packed(N, M), packed(K, M)
        s["dX"], s["dW"] = _empty(bf, M, K), _empty(bf, N, K)
    elif op == "quant":
        R, C = c["R"], c["C"]
        if c["axis"] != "columns":
            s["Xq"], s["V"] = packed(R, C, c["block"]), _empty(bf, R, C)
        if c["axis"] != "rows":
            s["Xt"], s["Vt"] = packed(C, R, c["block"]), _empty(bf, C, R)
    else:
        T, E, k = c["T"], c["E"], c["k"]
        if op == "route" and c["grad"]:
            s["dlogits_"] = _empty(f32, T, E)
        else:
            s["idx_"], s["w_"] = _empty(i32, T, k), _empty(f32, T, k)
        if op != "route":
            D, F, R = c["D"], c["F"], _slots(c)
            s["order"] = _empty(i32, 2 * E + 64 + T * k + R + R // 128)
            if op == "experts":
                s["Xq"], s["Hq"] = packed(T, D), packed(R, F)
                s["Y_"], s["out_"] = _empty(f32, R, D), _empty(bf, T, D)
            else:
                s["dYq"], s["dYt"], s["Ht"], s["Xt"] = packed(R, D), packed(D, R), packed(F, R), packed(D, R)
                s["dGUq"], s["dGUt"] = packed(R, 2 * F), packed(2 * F, R)
                s["dH_"], s["dXs_"], s["dX_"] = _empty(f32, R, F), _empty(f32, R, D), _empty(bf, T, D)
                s["dW1_"], s["dW2_"] = _empty(bf, E, 2 * F, D), _empty(bf, E, D, F)
                s["dw_"], s["dlogits_"] = _empty(f32, T, k), _empty(f32, T, E)
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
_SCORING = {"softmax": 0, "sigmoid": 1}


def _p(t):
    return None if t is None else t.data_ptr()


def _pp(pair):
    return pair[0].data_ptr(), pair[1].data_ptr()


def _own_route(ctx, c, s):
    groups = c.get("groups", 1)
    ctx.route_experts(_p(s["logits"]), _p(s.get("bias")), _p(s["idx_"]), _p(s["w_"]), c["T"], c["k"], c["E"],
                      scoring=_SCORING[c["scoring"]], groups=groups, groups_kept=c.get("kept", 1),
                      group_top=min(2, c["E"] // groups) if groups > 1 else 1, renormalize=True, scale=_SCALE)


def _run_own(s: dict):
    c, ctx = s["case"], _context()
    op = c["op"]
    if op == "linear":
        M, K, N = c["M"], c["K"], c["N"]
        xq = _pp(s["Xq"])
        ctx.quant_fp8(_p(s["X"]), M, K, *xq, dtype=_BF16)
        ctx.gemm_fp8(*xq, *_pp(s["W"]), _p(s["C"]), M, N, K, dtype=_BF16)
        return s["C"]
    if op == "gemm":
        ctx.gemm_fp8(*_pp(s["A"]), *_pp(s["B"]), _p(s["C"]), c["M"], c["N"], c["K"], dtype=_BF16)
        return s["C"]
    if op == "linear_grad":
        M, N, K = c["M"], c["N"], c["K"]
        dyq, dyt, xt = _pp(s["dYq"]), _pp(s["dYt"]), _pp(s["Xt"])
        ctx.quant_fp8(_p(s["dY"]), M, N, *dyq, *dyt, dtype=_BF16)
        ctx.quant_fp8(_p(s["X"]), M, K, None, None, *xt, dtype=_BF16)
        ctx.gemm_fp8(*dyq, *_pp(s["Wt"]), _p(s["dX"]), M, K, N, dtype=_BF16)
        ctx.gemm_fp8(*dyt, *xt, _p(s["dW"]), N, K, M, b_block=1, dtype=_BF16)
        return s["dX"], s["dW"]
    if op == "quant":
        R, C, X, block = c["R"], c["C"], s["X"], c["block"]
        q, qt = s.get("Xq"), s.get("Xt")
        ctx.quant_fp8(_p(X), R, C, *(_pp(q) if q else (None, None)), *(_pp(qt) if qt else (None, None)), block=block,
                      dtype=_CODE[X.dtype])
        out = []
        if q:
            ctx.dequant_fp8(*_pp(q), _p(s["V"]), R, C, block=block, dtype=_BF16)
            out.append(s["V"])
        if qt:
            ctx.dequant_fp8(*_pp(qt), _p(s["Vt"]), C, R, block=block, dtype=_BF16)
            out.append(s["Vt"])
        return out
    T, E, k = c["T"], c["E"], c["k"]
    if op == "route":
        if c["grad"]:
            ctx.route_experts_grad(_p(s["logits"]), _p(s["idx"]), _p(s["dw"]), _p(s["dlogits_"]), T, k, E,
                                   scoring=_SCORING[c["scoring"]], renormalize=True, scale=_SCALE)
            return s["dlogits_"]
        _own_route(ctx, c, s)
        return s["idx_"], s["w_"]
    D, F, order, n = c["D"], c["F"], _p(s["order"]), (T, k, E)
    if op == "experts":
        xq = _pp(s["Xq"])
        _own_route(ctx, c, s)
        ctx.experts_order(_p(s["idx_"]), order, *n)
        ctx.quant_fp8(_p(s["X"]), T, D, *xq, dtype=_BF16)
        ctx.experts_mlp_fp8(order, _p(s["w_"]), *xq, *_pp(s["W1"]), *_pp(s["W2"]), *_pp(s["Hq"]), _p(s["Y_"]),
                            _p(s["out_"]), *n, D, F, D, dtype=_BF16, y_dtype=_F32)
        return s["idx_"], s["w_"], s["out_"]
    dyq, dyt, dguq, dgut = _pp(s["dYq"]), _pp(s["dYt"]), _pp(s["dGUq"]), _pp(s["dGUt"])
    ht, xt, dh = _pp(s["Ht"]), _pp(s["Xt"]), _p(s["dH_"])
    ctx.experts_order(_p(s["idx"]), order, *n)
    ctx.experts_combine_grad(order, _p(s["Y"]), _p(s["dout"]), _p(s["dw_"]), *n, D, dtype=_BF16)
    ctx.route_experts_grad(_p(s["logits"]), _p(s["idx"]), _p(s["dw_"]), _p(s["dlogits_"]), T, k, E,
                           scoring=_SCORING[c["scoring"]], renormalize=True, scale=_SCALE)
    ctx.experts_quant_fp8(order, _p(s["dout"]), _p(s["w"]), *dyq, *dyt, *n, D, dtype=_BF16)
    ctx.experts_quant_fp8(order, _p(s["X"]), None, None, None, *xt, *n, D, dtype=_BF16)
    ctx.experts_gemm_fp8(order, *dyq, *_pp(s["W2t"]), dh, *n, F, D, dtype=_F32)
    ctx.experts_swiglu_fp8(order, _p(s["GU"]), None, None, *ht, *n, F, dtype=_BF16)
    ctx.experts_swiglu_grad_fp8(order, _p(s["GU"]), dh, *dguq, *dgut, *n, F, dtype=_BF16)
    ctx.experts_gemm_fp8(order, *dguq, *_pp(s["W1t"]), _p(s["dXs_"]), *n, D, 2 * F, dtype=_F32)
    ctx.experts_combine(order, _p(s["dXs_"]), None, _p(s["dX_"]), *n, D, dtype=_BF16, y_dtype=_F32)
    ctx.experts_wgrad_fp8(order, *dyt, *ht, _p(s["dW2_"]), *n, D, F, dtype=_BF16)
    ctx.experts_wgrad_fp8(order, *dgut, *xt, _p(s["dW1_"]), *n, 2 * F, D, dtype=_BF16)
    return s["dX_"], s["dW1_"], s["dW2_"], s["dlogits_"]


# ------------------------------------------------------------------ ... in plain form
def _power_of_two(amax: torch.Tensor) -> torch.Tensor:
    mantissa, exponent = torch.frexp(amax)  # 448 = 0.875 2^9
    return torch.ldexp(torch.ones_like(amax), (exponent - 9 + (mantissa > 0.875)).clamp(min=-126))


def _quantised(X: torch.Tensor, block: int, scale=_power_of_two):
    """(Q, S) of a matrix, along its rows."""
    R, K = X.shape
    x = torch.nn.functional.pad(X.float(), (0, _up(K) - K, 0, _up(R, block) - R))
    x = x.reshape(-1, block, _up(K) // 128, 128)
    S = scale(x.abs().amax((1, 3)))
    Q = (x / S[:, None, :, None]).to(torch.float8_e4m3fn)
    return Q.reshape(-1, _up(K))[:R].view(torch.uint8), S.t().contiguous()


def _transposed(W, rows, cols):
    """The packed transpose of packed weights (of every expert), which has the same elements and scales."""
    Q, S = W
    q = torch.nn.functional.pad(Q[..., :cols].transpose(-1, -2), (0, _up(rows) - rows))
    return q.contiguous(), S.transpose(-1, -2).contiguous()


def _values(Q: torch.Tensor, S: torch.Tensor, R: int, K: int, block: int = 128) -> torch.Tensor:
    """The fp32 values that a packed matrix stands for."""
    s = S.t().repeat_interleave(block, 0)[:R]
    return (Q.view(torch.float8_e4m3fn).float().reshape(R, -1, 128) * s.unsqueeze(-1)).reshape(R, -1)[:, :K]


def _rounded(X: torch.Tensor, block: int = 1) -> torch.Tensor:
    """X rounded to E4M3 along its rows."""
    return _values(*_quantised(X, block), *X.shape, block)


def _columns(X: torch.Tensor) -> torch.Tensor:
    return X.t().contiguous()


def _scores(c: dict, logits: torch.Tensor) -> torch.Tensor:
    """In 64 bits: two experts' scores may be next to each other."""
    l = logits.double()
    if c["scoring"] == "sigmoid":
        return 1 / (1 + torch.exp(-l))
    e = torch.exp(l - l.amax(-1, keepdim=True).clamp(min=-1e300))
    return e / e.sum(-1, keepdim=True).clamp(min=1e-300)


def _route(c: dict, s: dict):
    T, E, groups = c["T"], c["E"], c.get("groups", 1)
    score = _scores(c, s["logits"])
    choice = score + s["bias"].double() if "bias" in s else score
    choice = torch.where(s["logits"] == _NONE, _NONE, choice)
    if groups > 1:  # a group is as good as its best two experts
        best = choice.reshape(T, groups, -1).sort(-1, descending=True).values[..., :2]
        of = torch.where(best == _NONE, 0.0, best).sum(-1)
        of = torch.where(best[..., 0] == _NONE, _NONE, of)
        kept = torch.sort(of, dim=-1, descending=True, stable=True).indices[:, :c["kept"]]
        keep = torch.zeros(T, groups, dtype=torch.bool, device=score.device).scatter_(1, kept, True)
        choice = torch.where(keep.repeat_interleave(E // groups, 1), choice, _NONE)
    value, idx = torch.sort(choice, dim=-1, descending=True, stable=True)  # (of equals the lowest index first)
    value, idx = value[:, :c["k"]], idx[:, :c["k"]]
    w = torch.where(value == _NONE, 0.0, score.gather(1, idx))
    w = _SCALE * w / (w.sum(-1, keepdim=True) + 1e-20)
    return torch.where(value == _NONE, -1, idx).int(), w.float()


def _route_backward(c: dict, s: dict, dw: torch.Tensor):
    p, dw, some = _scores(c, s["logits"]).float(), dw.float(), s["idx"] >= 0
    at = s["idx"].clamp(min=0).long()
    chosen = torch.where(some, p.gather(1, at), 0.0)
    total = chosen.sum(-1, keepdim=True) + 1e-20
    dw = torch.where(some, dw, 0.0)
    ds = _SCALE * (dw - (dw * chosen).sum(-1, keepdim=True) / total) / total
    ds = torch.zeros_like(p).scatter_add_(1, at, torch.where(some, ds, 0.0))
    if c["scoring"] == "sigmoid":
        return ds * p * (1 - p)
    return p * (ds - (ds * p).sum(-1, keepdim=True))


def _swiglu(GU: torch.Tensor) -> torch.Tensor:
    g, u = GU.float().chunk(2, -1)
    return g / (1 + torch.exp(-g)) * u


def _run_plain(s: dict):
    c = s["case"]
    op = c["op"]
    if op == "linear":
        return (_rounded(s["X"]) @ _values(*s["W"], c["N"], c["K"]).t()).to(torch.bfloat16)
    if op == "gemm":
        A, B = _values(*s["A"], c["M"], c["K"], 1), _values(*s["B"], c["N"], c["K"])
        return (A @ B.t()).to(torch.bfloat16)
    if op == "linear_grad":
        dX = _rounded(s["dY"]) @ _values(*s["Wt"], c["K"], c["N"]).t()
        dW = _rounded(_columns(s["dY"])) @ _rounded(_columns(s["X"])).t()
        return dX.to(torch.bfloat16), dW.to(torch.bfloat16)
    if op == "quant":
        out = []
        if c["axis"] != "columns":
            out.append(_rounded(s["X"], c["block"]).to(torch.bfloat16))
        if c["axis"] != "rows":
            out.append(_rounded(_columns(s["X"]), c["block"]).to(torch.bfloat16))
        return out
    if op == "route":
        return _route_backward(c, s, s["dw"]) if c["grad"] else _route(c, s)
    return _experts(c, s) if op == "experts" else _experts_backward(c, s)


def _experts(c: dict, s: dict):
    D, F = c["D"], c["F"]
    idx, w = _route(c, s)
    X, out = _rounded(s["X"]), torch.zeros(c["T"], D, device="cuda")
    for e in range(c["E"]):
        mine = idx == e
        H = _rounded(_swiglu(X @ _values(s["W1"][0][e], s["W1"][1][e], 2 * F, D).t()))
        Y = H @ _values(s["W2"][0][e], s["W2"][1][e], D, F).t()
        out += torch.where(mine.any(-1, keepdim=True), Y, 0.0) * torch.where(mine, w, 0.0).sum(-1, keepdim=True)
    return idx, w, out.to(torch.bfloat16)


def _experts_backward(c: dict, s: dict):
    T, E, D, F = c["T"], c["E"], c["D"], c["F"]
    R, place = s["GU"].shape[0], torch.arange(T, device="cuda")
    dX, dw = torch.zeros(T, D, device="cuda"), torch.zeros(T, c["k"], device="cuda")
    dW1, dW2 = torch.zeros(E, 2 * F, D, device="cuda"), torch.zeros(E, D, F, device="cuda")
    for e in range(E):
        rows, some = s["row"][e], (place < s["count"][e]).unsqueeze(-1)  # this expert's tokens first, the others masked
        at = (s["start"][e] + place).clamp(max=R - 1)
        dout, GU, X = s["dout"][rows].float(), s["GU"][at], s["X"][rows].float() * some
        mine = (s["idx"][rows] == e) & some
        dw.index_add_(0, rows, torch.where(mine, (dout * s["Y"][at].float()).sum(-1, keepdim=True), 0.0))
        dY = dout * torch.where(mine, s["w"][rows], 0.0).sum(-1, keepdim=True)
        dH = _rounded(dY) @ _values(s["W2t"][0][e], s["W2t"][1][e], F, D).t()
        g, u = GU.float().chunk(2, -1)
        sig = 1 / (1 + torch.exp(-g))
        dGU = torch.cat((dH * u * sig * (1 + g * (1 - sig)), dH * g * sig), -1) * some
        dXe = _rounded(dGU) @ _values(s["W1t"][0][e], s["W1t"][1][e], D, 2 * F).t()
        dX.index_add_(0, rows, torch.where(some, dXe, 0.0))
        dW2[e] = _rounded(_columns(dY)) @ _rounded(_columns(_swiglu(GU) * some)).t()
        dW1[e] = _rounded(_columns(dGU)) @ _rounded(_columns(X)).t()
    return dX.to(torch.bfloat16), dW1.to(torch.bfloat16), dW2.to(torch.bfloat16), _route_backward(c, s, dw)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case: dict) -> dict:
    c, op = case, case["op"]
    if op in ("linear", "gemm"):
        M, N, K = c["M"], c["N"], c["K"]
        return {"bytes": (2 if op == "linear" else 1) * M * K + N * K + 2 * M * N,
                "flops": 2 * M * N * K}
    if op == "linear_grad":
        M, N, K = c["M"], c["N"], c["K"]
        return {"bytes": 2 * (M * N + M * K) + N * K + 2 * M * K + 2 * N * K, "flops": 4 * M * N * K}
    if op == "quant":  # the packed matrices, written once, and the values
        n, k = c["R"] * c["C"], 2 if c["axis"] == "both" else 1
        return {"bytes": (2 if c["dtype"] == "bf16" else 4) * n + 3 * k * n, "flops": 0}
    T, E, k = c["T"], c["E"], c["k"]
    routing = 4 * T * E + 8 * T * k
    if op == "route":
        return {"bytes": routing + (4 * T * E if c["grad"] else 0), "flops": 0}
    D, F = c["D"], c["F"]
    used = E * (1 - (1 - k / E)**T)  # experts that some token goes to, if all are liked as well
    n = (T - T // 10 if c["masked"] else T) * k
    if op == "experts":
        return {"bytes": int(used * 3 * D * F) + 4 * T * D + routing, "flops": 6 * n * D * F}
    saved = 2 * n * (2 * F + D)  # gate and up projections, outputs
    return {"bytes": int(used * 3 * D * F) + saved + 6 * T * D + 6 * E * D * F + 2 * routing, "flops": 12 * n * D * F}


# ------------------------------------------------------------------ the same in 64 bits
def _exact_values(Q, S, R, K, block=128):
    """Values of a packed matrix from the fields of its codes: sign, four exponent bits, three mantissa bits."""
    code = Q[:, :K].int()
    exponent, mantissa = (code >> 3) & 15, (code & 7).double()
    size = torch.where(exponent > 0, (8 + mantissa) * torch.exp2(exponent.double() - 10), mantissa * 2.0**-9)
    row, col = torch.arange(R, device=Q.device) // block, torch.arange(K, device=Q.device) // 128
    return torch.where(code >= 128, -size, size) * S.double()[col][:, row].t()


def _exact_rounded(X, block=1):
    """Each element to the nearest multiple of its binade's step, in units of its block's power of two."""
    R, K = X.shape
    x = X.double()
    amax = torch.nn.functional.pad(x.abs(), (0, -K % 128, 0, -R % block))
    amax = amax.reshape(-1, block, -(-K // 128), 128).amax((1, 3))
    scale = torch.exp2(torch.ceil(torch.log2((amax / 448).clamp(min=2.0**-126)))).repeat_interleave(block, 0)[:R].repeat_interleave(128, 1)[:, :K]
    a = x.abs() / scale
    step = torch.exp2(torch.floor(torch.log2(a.clamp(min=2.0**-6))) - 3)
    return torch.sign(x) * (torch.round(a / step) * step).clamp(max=448) * scale


def _exact_product(A, B):
    return A.contiguous() @ B.t().contiguous()


def exact(case: dict, seed: int):
    c, s = case, _inputs(case, seed)
    op = c["op"]
    if op == "linear":
        return _exact_product(_exact_rounded(s["X"]), _exact_values(*s["W"], c["N"], c["K"]))
    if op == "gemm":
        return _exact_product(_exact_values(*s["A"], c["M"], c["K"], 1), _exact_values(*s["B"], c["N"], c["K"]))
    if op == "linear_grad":
        dY, X = s["dY"].double(), s["X"].double()
        return (_exact_product(_exact_rounded(dY), _exact_values(*s["Wt"], c["K"], c["N"])),
                _exact_product(_exact_rounded(dY.t()), _exact_rounded(X.t())))
    if op == "quant":
        X = s["X"].double()
        return [_exact_rounded(m, c["block"]) for m, a in ((X, "columns"), (X.t(), "rows")) if c["axis"] != a]
    if op == "route":
        if c["grad"]:
            return _exact_route_grad(c, s["logits"], s["idx"], s["dw"].double())
        return _exact_route(c, s)
    return _exact_experts(c, s) if op == "experts" else _exact_experts_grad(c, s)


def _exact_scores(c, logits):
    """(a token of padding has no scores)"""
    some = torch.isfinite(logits).any(-1, keepdim=True)
    l = torch.where(some, logits, torch.zeros_like(logits))
    p = torch.sigmoid(l) if c["scoring"] == "sigmoid" else torch.softmax(l, -1)
    return torch.where(some, p, torch.zeros_like(p))


def _exact_weights(c, p, idx):
    """Weights of the chosen experts by token, differentiable in the scores p."""
    some = idx >= 0
    chosen = p.gather(1, idx.clamp(min=0).long()) * some
    return _SCALE * chosen / (chosen.sum(-1, keepdim=True) + 1e-20)


def _exact_route(c, s):
    """The best expert again and again, among the groups found alike."""
    T, E, groups = c["T"], c["E"], c.get("groups", 1)
    p = _exact_scores(c, s["logits"].double())
    left = p + s["bias"].double() if "bias" in s else p.clone()
    allowed = torch.isfinite(s["logits"])
    left = left.masked_fill(~allowed, -math.inf)
    if groups > 1:
        of = left.view(T, groups, E // groups).topk(min(2, E // groups), dim=-1).values
        of = torch.where(torch.isfinite(of[..., 0]), torch.nan_to_num(of, neginf=0.0).sum(-1), -math.inf)
        keep = torch.zeros(T, groups, dtype=torch.bool, device=p.device)
        for _ in range(c["kept"]):
            best = of.argmax(-1, keepdim=True)
            keep.scatter_(1, best, True)
            of = of.scatter(1, best, -math.inf)
        left = left.masked_fill(~keep.repeat_interleave(E // groups, 1), -math.inf)
    idx = torch.empty(T, c["k"], dtype=torch.int32, device=p.device)
    for j in range(c["k"]):
        top = left.amax(-1, keepdim=True)
        first = torch.where(left == top, torch.arange(E, device=p.device), E).amin(-1)
        idx[:, j] = torch.where(torch.isfinite(top[:, 0]), first, -1)
        left = left.scatter(1, first.unsqueeze(1), -math.inf)
    return idx, _exact_weights(c, p, idx)


def _exact_route_grad(c, logits, idx, dw):
    l = logits.double().requires_grad_()
    return torch.autograd.grad(_exact_weights(c, _exact_scores(c, l), idx), l, dw)[0].nan_to_num(0.0)


def _exact_swiglu(gate, up):
    return gate * torch.sigmoid(gate) * up


def _exact_experts(c, s):
    idx, w = _exact_route(c, s)
    D, F = c["D"], c["F"]
    X, out = _exact_rounded(s["X"]), torch.zeros(c["T"], D, dtype=torch.float64, device="cuda")
    for e in range(c["E"]):
        token, choice = torch.nonzero(idx == e, as_tuple=True)
        GU = _exact_product(X[token], _exact_values(s["W1"][0][e], s["W1"][1][e], 2 * F, D))
        Y = _exact_product(_exact_rounded(_exact_swiglu(GU[:, :F], GU[:, F:])),
                           _exact_values(s["W2"][0][e], s["W2"][1][e], D, F))
        out.index_add_(0, token, Y * w[token, choice].unsqueeze(-1))
    return idx, w, out


def _exact_experts_grad(c, s):
    T, E, D, F = c["T"], c["E"], c["D"], c["F"]

    def zeros(*shape):
        return torch.zeros(shape, dtype=torch.float64, device="cuda")

    dX, dw, dW1, dW2 = zeros(T, D), zeros(T, c["k"]), zeros(E, 2 * F, D), zeros(E, D, F)
    for e in range(E):
        token, choice = torch.nonzero(s["idx"] == e, as_tuple=True)  # (in the order of the tokens)
        if len(token) == 0:
            continue
        at = slice(int(s["start"][e]), int(s["start"][e]) + len(token))
        dout, X = s["dout"][token].double(), s["X"][token].double()
        dw[token, choice] = (dout * s["Y"][at].double()).sum(-1)
        dY = dout * s["w"][token, choice].double().unsqueeze(-1)
        gate = s["GU"][at, :F].double().requires_grad_()
        up = s["GU"][at, F:].double().requires_grad_()
        H = _exact_swiglu(gate, up)
        dH = _exact_product(_exact_rounded(dY), _exact_values(s["W2t"][0][e], s["W2t"][1][e], F, D))
        dGU = torch.cat(torch.autograd.grad(H, (gate, up), dH), -1)
        dX.index_add_(0, token, _exact_product(_exact_rounded(dGU), _exact_values(s["W1t"][0][e], s["W1t"][1][e], D, 2 * F)))
        dW2[e] = _exact_product(_exact_rounded(dY.t()), _exact_rounded(H.detach().t()))
        dW1[e] = _exact_product(_exact_rounded(dGU.t()), _exact_rounded(X.t()))
    return dX, dW1, dW2, _exact_route_grad(c, s["logits"], s["idx"], dw)
