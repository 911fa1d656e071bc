"""What is measured of the 8-bit integer linear layer: the RMS norm and the row quantiser that make int8 rows with a
scale for each row (token), and the int8 product with scales for each row and each output channel.

The sizes are the evaluator's own: rows are tokens (65 a board, 66,560 for a batch of 1,024 boards, 1 for a single
CLS row), widths the network's d = 1,024 and feed-forward 2,048, 8,324 the two heads; others are generic.

Int8 rows are returned as the values they stand for (code times scale, rounded to bf16), beside their scales.
"""
import math

import torch

own = False

_DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_SIZE = {"f32": 4, "bf16": 2, "f16": 2}
_EPS = 1e-6
_ROWS = 66560                      # 1,024 boards of 65 tokens
_MOST = _ROWS * 2048               # elements of the largest activation
_MACS = _ROWS * 2048 * 1024        # multiply-adds of the largest product


def listed():
    return [
        # one token's residual row before a product: the smallest call, all latency
        {"name": "norm_1x1024", "op": "norm", "M": 1, "D": 1024, "x": "f32", "delta": "bf16"},
        # eight boards of a network whose width is no multiple of anything
        {"name": "norm_520x997_f16", "op": "norm", "M": 520, "D": 997, "x": "f16", "delta": "f16"},
        # a wide bf16 residual stream
        {"name": "norm_4097x8192_bf16", "op": "norm", "M": 4097, "D": 8192, "x": "bf16", "delta": "bf16"},
        # 1,024 boards: the f32 residual stream and a product's bf16 output added to it
        {"name": "norm_66560x1024", "op": "norm", "M": _ROWS, "D": 1024, "x": "f32", "delta": "bf16"},
        # one board's feed-forward activations before the second product
        {"name": "quant_65x2048", "op": "quant", "M": 65, "D": 2048, "x": "bf16"},
        # the heads' weights, a scale for each output channel
        {"name": "quant_8324x1024_f32", "op": "quant", "M": 8324, "D": 1024, "x": "f32"},
        # 1,024 boards' feed-forward activations
        {"name": "quant_66560x2048", "op": "quant", "M": _ROWS, "D": 2048, "x": "bf16"},
        # both heads of one board: one row against 8,324 channels
        {"name": "gemm_1x8324x1024", "op": "gemm", "M": 1, "N": 8324, "K": 1024, "epi": 3, "out": "f32", "bias": True},
        # one board's first feed-forward product
        {"name": "gemm_65x2048x1024_gelu", "op": "gemm", "M": 65, "N": 2048, "K": 1024, "epi": 1, "out": "bf16",
         "bias": True},
        # a few tokens against a large weight: the weight's bytes are the work
        {"name": "gemm_16x8192x8192", "op": "gemm", "M": 16, "N": 8192, "K": 8192, "epi": 0, "out": "bf16",
         "bias": False},
        # odd sizes, added into an f32 residual stream
        {"name": "gemm_777x1001x1000_add", "op": "gemm", "M": 777, "N": 1001, "K": 1000, "epi": 2, "out": "f32",
         "bias": True},
        # 1,024 boards' first feed-forward product
        {"name": "gemm_66560x2048x1024_gelu", "op": "gemm", "M": _ROWS, "N": 2048, "K": 1024, "epi": 1, "out": "bf16",
         "bias": True},
    ]


def _log(rng, lo, hi):
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if rng.random() < 0.5 and n >= 256:      # half of the larger sizes whole multiples of 64, the others as they fall
        n -= n % 64
    return max(lo, min(hi, n))


def draw(rng):
    op = rng.choice(["norm", "quant", "gemm"])
    while True:
        M = _log(rng, 1, _ROWS)
        if op == "gemm":
            N, K, epi = _log(rng, 64, 8324), _log(rng, 64, 8192), rng.choice([0, 1, 2, 3])
            if M * N * K > _MACS or M * N > _MOST or M * K > _MOST:
                continue
            return {"op": op, "M": M, "N": N, "K": K, "epi": epi,
                    "out": rng.choice(["bf16", "f16"]) if epi < 2 else "f32", "bias": rng.random() < 0.75}
        D = _log(rng, 64, 8192)
        if op == "quant":
            if M * D <= _MOST:
                return {"op": op, "M": M, "D": D, "x": rng.choice(["f32", "bf16", "f16"])}
        elif M * D <= _ROWS * 1024:
            x = rng.choice(["f32", "bf16", "f16"])
            delta = rng.choice(["f32", "bf16", "f16", "none"] if x == "f32" else [x, x, "none"])
            return {"op": op, "M": M, "D": D, "x": x, "delta": delta}


def _pitch(n):
    return -(-n // 16) * 16          # int8 rows of a product's operand begin on 16 bytes


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    M = case["M"]
    randn = lambda *n: torch.randn(*n, device="cuda", generator=g)  # noqa: E731
    rand = lambda *n: torch.rand(*n, device="cuda", generator=g)  # noqa: E731
    s = {"case": case}
    if case["op"] == "gemm":
        N, K = case["N"], case["K"]
        code = lambda r: torch.zeros(r, _pitch(K), dtype=torch.int8, device="cuda")  # noqa: E731
        for name, r in (("A", M), ("W", N)):
            t = code(r)
            # what quantising a normal row gives: the largest of the row at 127, one sigma near 36
            t[:, :K] = (randn(r, K) * 36).round().clamp(-127, 127).to(torch.int8)
            s[name] = t[:, :K]
        s["rowscale"] = (rand(M) + 0.5) / 36
        s["colscale"] = (rand(N) + 0.5) / (36 * math.sqrt(K))
        s["bias"] = randn(N) * 0.02 if case["bias"] else None
        s["C"] = randn(M, N) if case["epi"] == 2 else torch.empty(M, N, dtype=_DT[case["out"]], device="cuda")
        return s
    D, dt = case["D"], _DT[case["x"]]
    # activations: a few channels far larger than the rest
    channel = torch.where(rand(D) < 0.01, 8.0, 1.0)
    s["x"] = (randn(M, D) * channel).to(dt)
    s["q"] = torch.zeros(M, _pitch(D), dtype=torch.int8, device="cuda")[:, :D]
    s["scale"] = torch.empty(M, device="cuda")
    s["column"] = s["scale"][:, None]
    s["values"] = torch.empty(M, D, dtype=torch.bfloat16, device="cuda")
    if case["op"] == "norm":
        s["delta"] = (randn(M, D) * 0.5).to(_DT[case["delta"]]) if case["delta"] != "none" else None
        s["g"] = 1 + 0.1 * randn(D)
        s["out"] = torch.empty_like(s["x"]) if case["delta"] != "none" else None
    return s


# ---------------------------------------------------------------- the plain forms
def _codes(t):
    """Rows of t as whole numbers -127..127, and max |t| of each row."""
    a = t.abs().amax(1, keepdim=True)
    zero = a < 2.0 ** -120
    return torch.where(zero, torch.zeros_like(t), torch.round(t * (127.0 / torch.where(zero, torch.ones_like(a), a)))), a


def _plain_norm(s):
    x = s["x"]
    if s["delta"] is not None:
        x = (x.float() + s["delta"].float()).to(x.dtype)
    h = x.float()
    r = torch.rsqrt(h.square().mean(1, keepdim=True) + _EPS)
    q, a = _codes(h * s["g"])
    scale = a * r / 127.0
    return [x if s["delta"] is not None else None, (q * scale).to(torch.bfloat16), scale[:, 0]]


def _plain_quant(s):
    q, a = _codes(s["x"].float())
    scale = a / 127.0
    return [(q * scale).to(torch.bfloat16), scale[:, 0]]


def _plain_gemm(s):
    epi, C = s["case"]["epi"], s["C"]
    # products of int8 codes: whole numbers, whose sums float32 holds exactly up to 2^24
    v = (s["A"].float() @ s["W"].float().t()) * s["rowscale"][:, None] * s["colscale"]
    if s["bias"] is not None:
        v = v + s["bias"]
    if epi == 2:
        C += v
        return C
    if epi == 1:
        v = 0.5 * v * (1 + torch.erf(v * math.sqrt(0.5)))
    return v.to(C.dtype)


# ---------------------------------------------------------------- the framework's operators
_k = None


def _kernels():
    global _k
    if _k is None:
        from mayfly_chess_b200 import cudanet_py
        _k = cudanet_py
    return _k


def _own(s):
    k = _k or _kernels()
    op = s["case"]["op"]
    if op == "gemm":
        return k.k_gemm_i8(s["A"], s["W"], s["rowscale"], s["colscale"], s["bias"], s["C"], s["case"]["epi"])
    if op == "norm":
        k.k_rmsnorm_i8(s["x"], s["delta"], s["g"], s["out"], s["q"], s["scale"], _EPS)
        first = [s["out"]]
    else:
        k.k_quant_i8(s["x"], s["q"], s["scale"])
        first = []
    return first + [torch.mul(s["q"], s["column"], out=s["values"]), s["scale"]]


def run(state):
    if own:
        return _own(state)
    return {"norm": _plain_norm, "quant": _plain_quant, "gemm": _plain_gemm}[state["case"]["op"]](state)


def work(case):
    M = case["M"]
    if case["op"] == "gemm":
        N, K = case["N"], case["K"]
        size = _SIZE[case["out"]] * (2 if case["epi"] == 2 else 1)     # read and written where it is added to
        return {"bytes": M * K + N * K + M * N * size + 4 * M + 4 * N * (2 if case["bias"] else 1),
                "flops": 2 * M * N * K}
    D, x = case["D"], _SIZE[case["x"]]
    if case["op"] == "quant":
        return {"bytes": M * D * (x + 1) + 4 * M, "flops": 3 * M * D}
    delta = _SIZE[case["delta"]] + x if case["delta"] != "none" else 0   # the sum is written too
    return {"bytes": M * D * (x + delta + 1) + 4 * M + 4 * D, "flops": 7 * M * D}


# ---------------------------------------------------------------- the definition in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    d = torch.float64
    if case["op"] == "gemm":
        y = torch.einsum("mk,nk->mn", s["A"].to(d), s["W"].to(d))
        y *= torch.outer(s["rowscale"].to(d), s["colscale"].to(d))
        if s["bias"] is not None:
            y += s["bias"].to(d)
        if case["epi"] == 1:
            y = y * torch.special.ndtr(y)
        if case["epi"] == 2:
            y += s["C"].to(d)
        return y
    head, y = [], s["x"].to(d)
    if case["op"] == "norm":
        if s["delta"] is not None:
            y += s["delta"].to(d)
            head = [y.clone()]
            # the norm is of the residual stream as it is stored
            y = y.to(_DT[case["x"]]).to(d)
        else:
            head = [None]
        rms = (torch.linalg.vector_norm(y, dim=1).square() / case["D"] + _EPS).sqrt()
        y = y * s["g"].to(d) / rms[:, None]
    scale = torch.linalg.vector_norm(y, ord=math.inf, dim=1) / 127
    codes = (y / scale[:, None]).round_()
    return head + [codes * scale[:, None], scale]
