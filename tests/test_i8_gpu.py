"""The int8 linear layer (k_rmsnorm_i8, k_quant_i8, k_gemm_i8) on a B200 against its definition in 64 bits.

Tolerances count the roundings between the definition and the result, u = 2^-24 each (half a step of f32, relative):
  codes    t * (127 / a) has a rounding in the factor and one in the product (for the norm one in t = s * g and one in
           a too), and is at most 127: off by 127 * 4u at most before it is rounded to a whole number, so a code is
           within 0.5 + 127 * 4u of the exact quotient
  scale    quantiser: one division, exactly the f32 quotient. Norm: a sum of squares of D terms, each thread at most
           D / 32 of them one after another and then a tree of at most 10 adds, each rounding at most u; the square
           root halves that; rsqrtf is within 2 steps (4u), and the mean, eps, t, a * r and the quotient are 5 more
  product  acc is exact; its conversion, two scalings and the bias are 4 roundings: 2u of |acc rs cs| and u of the
           result, and twice that bounds them; the 16-bit output adds eps / 2 of its type, GELU the relative
           error of Phi(-a) of its polynomial (2.5e-5 for f16, 2.6e-4 for bf16) times a * Phi(-a), which is at most
           0.17, and its slope of at most 1.13
These bounds of the codes and of the bf16 GELU are wider than what the kernels hold: test_codes_are_the_rounded_quotient,
test_rows_of_every_width (which counts the squares that a thread adds by its elements) and test_gelu_of_every_size have
their own.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


@pytest.fixture(scope="module")
def k():
    from mayfly_chess_b200 import build, cudanet_py
    build.build()
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return cudanet_py


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def matrix(rows, cols, dtype, pitch=None, fill=0, offset=0):
    """A (rows, cols) view, `offset` elements into a buffer of rows of `pitch` that is filled with `fill`, two rows more
    than the view's; and the buffer."""
    pitch = cols if pitch is None else pitch
    full = torch.full(((rows + 2) * pitch + offset,), fill, dtype=dtype, device="cuda")
    return full[offset:].view(rows + 2, pitch)[:rows, :cols], full


def untouched(view, full, fill, offset=0):
    """Whether nothing outside the view was written."""
    keep = full.clone()
    rows, cols = view.shape
    keep[offset:].view(rows + 2, -1)[:rows, :cols] = fill
    want = torch.full_like(full, fill)
    return torch.equal(keep.view(torch.uint8), want.view(torch.uint8))


def row_scale(x):
    """max |row| / 127 in f32: the quotient in 64 bits (of two tensors: torch multiplies by a number's reciprocal),
    which has more than twice f32's bits, rounded once."""
    a = x.double().abs().amax(1)
    return (a / torch.full_like(a, 127)).float()


def check_codes(q, scale, t64, scale64, scale_tol):
    """q and scale against the exact t (up to a row factor) and scale; every row here has something to scale."""
    a = t64.abs().amax(1, keepdim=True)
    assert ((scale.double() - scale64).abs() <= scale_tol * scale64).all()
    assert ((q.double() - 127 * t64 / a).abs() <= 0.5 + 127 * 4 * U).all()
    assert (q.abs().amax(1) == 127).all()


# ------------------------------------------------------------------------------------------------ rows
SHAPES = [(1, 1), (1, 1024), (3, 7), (5, 8), (2, 31), (65, 256), (66, 997), (7, 1000), (33, 1024), (4, 2048), (3, 4104),
          (2, 8191), (5, 8192), (2, 20001), (1, 32768), (3, 32760), (1300, 1024), (600, 72)]


@pytest.mark.parametrize("M,D", SHAPES)
@pytest.mark.parametrize("x", ["f32", "bf16", "f16"])
def test_quant(k, M, D, x):
    g = gen(M * 31 + D)
    X = (torch.randn(M, D, device="cuda", generator=g) * 3).to(DT[x])
    X[:, 0] = 1.0                      # no row of zeros
    q, scale = torch.empty(M, D, dtype=torch.int8, device="cuda"), torch.empty(M, device="cuda")
    assert k.k_quant_i8(X, q, scale) == (q, scale)
    t = X.double()
    assert torch.equal(scale, row_scale(X))
    check_codes(q, scale, t, t.abs().amax(1) / 127, U)


@pytest.mark.parametrize("M,D", SHAPES)
@pytest.mark.parametrize("x,delta", [("f32", "f32"), ("f32", "bf16"), ("f32", "f16"), ("f32", None), ("bf16", "bf16"),
                                     ("bf16", None), ("f16", "f16"), ("f16", None)])
def test_rmsnorm(k, M, D, x, delta):
    r = gen(M * 37 + D)
    X = torch.randn(M, D, device="cuda", generator=r).to(DT[x])
    X[:, 0] = 4.0
    G = 1 + 0.1 * torch.randn(D, device="cuda", generator=r)
    Dl = torch.randn(M, D, device="cuda", generator=r).to(DT[delta]) if delta else None
    want = X if delta is None else (X.float() + Dl.float()).to(X.dtype)
    out = torch.empty_like(X) if delta else None
    X0 = X.clone()
    q, scale = torch.empty(M, D, dtype=torch.int8, device="cuda"), torch.empty(M, device="cuda")
    k.k_rmsnorm_i8(X, Dl, G, out, q, scale, 1e-5)
    if delta:
        assert torch.equal(out, want) and torch.equal(X, X0)
    s = want.double()
    t = s * G.double()
    scale64 = t.abs().amax(1) / torch.sqrt(s.square().mean(1) + float(torch.tensor(1e-5))) / 127
    check_codes(q, scale, t, scale64, ((D / 32 + 10) / 2 + 9) * U)
    if delta:                          # in place, the same bits
        q2, scale2 = torch.empty_like(q), torch.empty_like(scale)
        k.k_rmsnorm_i8(X, Dl, G, X, q2, scale2, 1e-5)
        assert torch.equal(X, want) and torch.equal(q2, q) and torch.equal(scale2, scale)


@pytest.mark.parametrize("D,off", [(64, 0), (2048, 0), (999, 1)])
@pytest.mark.parametrize("x,low,high", [("f32", -119, 125), ("bf16", -119, 125), ("f16", -20, 13)])
def test_codes_at_the_ends_of_the_range(k, x, low, high, D, off):
    """Rows whose largest comes near the least that is scaled (or f16's least) and near the type's greatest."""
    e = torch.arange(low, high + 1, device="cuda")
    r = gen(D)
    base = torch.randn(len(e), D, device="cuda", generator=r).clamp(-3.9, 3.9)
    base[:, 1], base[:, D - 1] = 2.0, -1.0
    X, _ = matrix(len(e), D, DT[x], D, 0, off)
    X.copy_(torch.ldexp(base.to(DT[x]).double(), e[:, None]))
    q, scale = torch.empty(len(e), D, dtype=torch.int8, device="cuda"), torch.empty(len(e), device="cuda")
    k.k_quant_i8(X, q, scale)
    t = X.double()
    assert torch.equal(scale, row_scale(X)) and (scale > 0).all()
    assert torch.equal(q.float(), torch.round((127 * t / t.abs().amax(1, keepdim=True)).float()))


# A width on each side of every border between two row kernels, aligned and element by element, rows that leave part of a
# block or of a warp without one.
WIDTHS = [(M, D, off) for M, D in ((7, 8), (7, 64), (131, 72), (13, 128), (131, 136), (5, 256), (131, 264), (6, 512), (131, 520),
                                   (5, 768), (131, 776), (6, 1024), (131, 1032), (5, 1288), (131, 1536), (5, 1544),
                                   (131, 2048), (3, 2056), (3, 16384), (3, 16392), (2, 32768)) for off in (0, 1)]
WIDTHS += [(M, D, 1) for M, D in ((131, 1), (7, 65), (131, 129), (7, 257), (131, 511), (7, 513), (131, 600), (5, 767),
                                  (131, 769), (5, 1023), (131, 1025), (5, 2047), (5, 2049), (3, 16383), (3, 16385), (2, 32767))]


@pytest.mark.parametrize("M,D,off", WIDTHS)
@pytest.mark.parametrize("x,delta", [("f32", "f32"), ("f32", "bf16"), ("f32", "f16"), ("f32", None), ("bf16", "bf16"),
                                     ("bf16", None), ("f16", "f16"), ("f16", None)])
def test_rows_of_every_width(k, M, D, off, x, delta):
    """Codes of the norm as of test_rmsnorm. Its scale: at most 32 squares in a thread and 10 sums over warp and block,
    42u, halved by the root; the mean and eps u together after it, rsqrtf 4u, the largest, its product and the quotient
    u each: 29u, and 1u for products of these. Where the norm adds nothing, the quantiser of the same rows too."""
    r = gen(M * 41 + D)
    X, _ = matrix(M, D, DT[x], (D + 7) // 8 * 8 if off == 0 else D, 9, off)
    X.copy_(torch.randn(M, D, device="cuda", generator=r))
    X[:, D // 2] = 4.0
    G = 1 + 0.1 * torch.randn(D, device="cuda", generator=r)
    Dl = torch.randn(M, D, device="cuda", generator=r).to(DT[delta]) if delta else None
    want = X if delta is None else (X.float() + Dl.float()).to(X.dtype)
    out = torch.empty(M, D, dtype=X.dtype, device="cuda") if delta else None
    q, fq = matrix(M, D, torch.int8, (D + 15) // 16 * 16, 99)
    scale = torch.full((M + 1,), 9.0, device="cuda")
    k.k_rmsnorm_i8(X, Dl, G, out, q, scale[:M], 1e-5)
    if delta:
        assert torch.equal(out, want)
    s = want.double()
    t = (want.float() * G).double()
    scale64 = (s * G.double()).abs().amax(1) / torch.sqrt(s.square().mean(1) + float(torch.tensor(1e-5))) / 127
    check_codes(q, scale[:M], s * G.double(), scale64, 30 * U)
    assert torch.equal(q.float(), torch.round((127 * t / t.abs().amax(1, keepdim=True)).float()))
    assert untouched(q, fq, 99) and scale[M] == 9
    if delta is None:
        k.k_quant_i8(X, q, scale[:M])
        assert torch.equal(scale[:M], row_scale(X))
        assert torch.equal(q.float(), torch.round((127 * s / s.abs().amax(1, keepdim=True)).float()))
        assert untouched(q, fq, 99) and scale[M] == 9


@pytest.mark.parametrize("x", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("D,px,pd,po,pq,off", [(64, 64, 80, 72, 64, 0), (64, 65, 66, 67, 68, 1), (1000, 1008, 1000, 1001, 1008, 0),
                                               (100, 112, 104, 108, 112, 3), (2048, 2056, 2049, 2048, 2064, 8)])
def test_rows_of_any_pitch_and_start(k, x, D, px, pd, po, pq, off):
    """Every pitch and start gives the bits of the contiguous call, and nothing outside the rows is written."""
    M, r = 37, gen(D + px)
    X0 = torch.randn(M, D, device="cuda", generator=r).to(DT[x])
    D0 = torch.randn(M, D, device="cuda", generator=r).to(DT[x])
    G = torch.randn(D + 1, device="cuda", generator=r)[1:]
    want = [torch.empty_like(X0), torch.empty(M, D, dtype=torch.int8, device="cuda"), torch.empty(M, device="cuda")]
    k.k_rmsnorm_i8(X0, D0, G, *want)
    X, _ = matrix(M, D, DT[x], px, 9, off)
    Dl, _ = matrix(M, D, DT[x], pd, 9, off)
    out, fo = matrix(M, D, DT[x], po, 9, off)
    q, fq = matrix(M, D, torch.int8, pq, 99, off)
    scale = torch.full((M + 2,), 9.0, device="cuda")
    X.copy_(X0)
    Dl.copy_(D0)
    k.k_rmsnorm_i8(X, Dl, G, out, q, scale[1:-1])
    assert torch.equal(out, want[0]) and torch.equal(q, want[1])
    # the sum of squares may be added in another order for rows that are read in another way
    assert ((scale[1:-1] - want[2]).abs() <= (D / 32 + 10) * U * want[2]).all()
    assert untouched(out, fo, 9, off) and untouched(q, fq, 99, off) and scale[0] == 9 and scale[-1] == 9
    qq, fq = matrix(M, D, torch.int8, pq, 99, off)
    k.k_quant_i8(X, qq, scale[1:-1])
    assert torch.equal(scale[1:-1], row_scale(X0))
    check_codes(qq, scale[1:-1], X0.double(), X0.double().abs().amax(1) / 127, U)
    assert untouched(qq, fq, 99, off)


@pytest.mark.parametrize("x", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("M,D,pitch,off", [(3000, 1024, 1024, 0), (3000, 72, 80, 0), (2500, 727, 727, 1), (4000, 37, 37, 0),
                                           (700, 4001, 4001, 3), (600, 8192, 8192, 0), (100, 20000, 20000, 0)])
def test_sum_in_place(k, x, M, D, pitch, off):
    """The sum stored over x and over delta, where rows share 32-byte sectors with their neighbours too: the bits of the
    call that stores it elsewhere."""
    r = gen(M + D)
    X0 = torch.randn(M, D, device="cuda", generator=r).to(DT[x])
    D0 = torch.randn(M, D, device="cuda", generator=r).to(DT[x])
    G = 1 + 0.1 * torch.randn(D, device="cuda", generator=r)
    (X, fx), (Dl, fd), (out, _) = (matrix(M, D, DT[x], pitch, 9, off) for _ in range(3))
    X.copy_(X0)
    Dl.copy_(D0)
    q, scale = torch.empty(M, D, dtype=torch.int8, device="cuda"), torch.empty(M, device="cuda")
    k.k_rmsnorm_i8(X, Dl, G, out, q, scale)
    assert torch.equal(out, (X0.float() + D0.float()).to(DT[x])) and torch.equal(X, X0) and torch.equal(Dl, D0)
    for place, full in ((X, fx), (Dl, fd)):
        q2, scale2 = torch.empty_like(q), torch.empty_like(scale)
        X.copy_(X0)
        Dl.copy_(D0)
        k.k_rmsnorm_i8(X, Dl, G, place, q2, scale2)
        assert torch.equal(place, out) and torch.equal(q2, q) and torch.equal(scale2, scale)
        assert untouched(place, full, 9, off)


@pytest.mark.parametrize("D", [1, 33, 1024, 9000])
@pytest.mark.parametrize("x", ["f32", "bf16", "f16"])
def test_rows_with_nothing_to_scale(k, D, x):
    """Zero rows, rows of numbers too small to scale, and rows that hold a NaN or an infinity, among ordinary rows."""
    inf, nan = math.inf, math.nan
    X = torch.randn(10, D, device="cuda").to(DT[x])
    X[:, 0] = 2.0
    X[1] = 0.0
    X[2, D // 2] = nan
    X[3, D - 1] = inf
    X[4, D // 3] = -inf
    X[5] = -0.0
    X[6, 0], X[6, D - 1] = inf, nan
    if x != "f16":
        X[7] = 1e-38
    q, scale = torch.full((10, D), 99, dtype=torch.int8, device="cuda"), torch.full((10,), 9.0, device="cuda")
    k.k_quant_i8(X, q, scale)
    fine = [0, 8, 9] + ([7] if x == "f16" else [])
    zero = [1, 5] + ([] if x == "f16" else [7])
    assert torch.equal(scale[fine], row_scale(X[fine]))
    assert (scale[zero] == 0).all() and (q[zero] == 0).all()
    assert torch.isnan(scale[[2, 3, 4, 6]]).all() and (q[[2, 3, 4, 6]] == 0).all()
    G = torch.ones(D, device="cuda")
    q.fill_(99)
    k.k_rmsnorm_i8(X, None, G, None, q, scale)
    assert (scale[fine] > 0).all() and (q[fine].abs().amax(1) == 127).all()
    assert (scale[zero] == 0).all() and (q[zero] == 0).all()
    assert torch.isnan(scale[[2, 3, 4, 6]]).all() and (q[[2, 3, 4, 6]] == 0).all()
    if x != "f16":                      # squares over f32
        X.fill_(3e38)
        k.k_rmsnorm_i8(X, None, G, None, q, scale)
        assert torch.isnan(scale).all() and (q == 0).all()
    G.zero_()                           # a norm whose weight is zero
    k.k_rmsnorm_i8(X[:1].clone().fill_(1.0), None, G, None, q[:1], scale[:1])
    assert scale[0] == 0 and (q[0] == 0).all()


def test_codes_at_the_ties(k):
    """A row whose largest is 127 has the factor 1: its codes are its values rounded to the nearest, ties to even."""
    X = torch.arange(-127, 127.5, 0.5, device="cuda")[None].contiguous()
    q, scale = torch.empty(X.shape, dtype=torch.int8, device="cuda"), torch.empty(1, device="cuda")
    k.k_quant_i8(X, q, scale)
    assert scale[0] == 1 and torch.equal(q.float(), torch.round(X))


@pytest.mark.parametrize("x", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("D,off", [(8, 0), (8, 1), (727, 1), (1024, 0), (2048, 0), (2048, 1), (4104, 0)])
def test_codes_of_half_the_largest(k, x, D, off):
    """Half of a row's largest is 63.5 steps, a tie, whatever the largest is: code 64, the even one. Here the largest
    takes every bf16 mantissa."""
    a = ((1 + torch.arange(128, device="cuda") / 128) * 2.0 ** (torch.arange(128, device="cuda") % 9 - 4))[:, None]
    sign = torch.where(torch.arange(D, device="cuda") % 3 == 0, -1.0, 1.0)
    X, _ = matrix(128, D, DT[x], D, 0, off)
    X.copy_(sign * a / 2)
    X[:, D // 2] = a[:, 0].to(DT[x])
    want = 64 * sign.expand(128, D).clone()
    want[:, D // 2] = 127
    q, scale = torch.empty(128, D, dtype=torch.int8, device="cuda"), torch.empty(128, device="cuda")
    k.k_quant_i8(X, q, scale)
    assert torch.equal(q.float(), want)
    k.k_rmsnorm_i8(X, None, torch.ones(D, device="cuda"), None, q, scale)
    assert torch.equal(q.float(), want)


@pytest.mark.parametrize("x", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("M,D,off", [(2000, 2048, 0), (1000, 1001, 0), (300, 8192, 0), (5000, 130, 1)])
def test_codes_are_the_rounded_quotient(k, x, M, D, off):
    """A code is 127 t / max |t| in f32, rounded to a whole number, ties to even. In 64 bits the quotient has 29 bits
    more than it is then rounded to."""
    X, _ = matrix(M, D, DT[x], D, 0, off)
    X.copy_(torch.randn(M, D, device="cuda", generator=gen(D)))
    q, scale = torch.empty(M, D, dtype=torch.int8, device="cuda"), torch.empty(M, device="cuda")
    k.k_quant_i8(X, q, scale)
    t = X.double()
    assert torch.equal(q.float(), torch.round((127 * t / t.abs().amax(1, keepdim=True)).float()))


# ------------------------------------------------------------------------------------------------ product
def operands(M, N, K, seed, full=False):
    """Codes whose rows begin on 16 bytes, what lies behind them filled with codes that must not count."""
    r = gen(seed)
    pitch = (K + 15) // 16 * 16 + 16
    A, _ = matrix(M, K, torch.int8, pitch, 77)
    W, _ = matrix(N, K, torch.int8, pitch, -99)
    for t in (A, W):
        t.copy_(torch.randint(-128, 128, t.shape, device="cuda", generator=r, dtype=torch.int32).to(torch.int8))
    rs = (torch.rand(M, device="cuda", generator=r) + 0.5) / 64
    cs = (torch.rand(N, device="cuda", generator=r) + 0.5) / (64 * math.sqrt(K))
    bias = torch.randn(N, device="cuda", generator=r) * 0.1
    return A, W, rs, cs, bias


def check_product(C, C0, A, W, rs, cs, bias, epi):
    acc = A.double() @ W.double().t()                # whole numbers below 2^53: exact
    p = acc * rs.double()[:, None] * cs.double()
    v = p if bias is None else p + bias.double()
    tol = 2 * (2 * U * p.abs() + U * v.abs())
    if epi == 1:
        v = v * torch.special.ndtr(v)
        tol = 1.13 * tol + (2.6e-4 if C.dtype == torch.bfloat16 else 2.5e-5) * 0.17 + 4 * U * v.abs()
    if epi == 2:
        v = v + C0.double()
        tol = tol + U * v.abs()
    if epi < 2:
        f = torch.finfo(C.dtype)
        tol = tol + (v.abs() + tol) * f.eps / 2 + f.smallest_normal * f.eps / 2
    excess = ((C.double() - v).abs() - tol).max().item()
    assert math.isfinite(excess) and excess <= 0, excess


KERNELS = (-1, 1, 2, 3, 4, 6, 10)      # the choice of the library and each of its kernels: all give the same bits
SIZES = [(1, 1, 1), (1, 8324, 1024), (2, 7, 15), (3, 64, 16), (5, 129, 130), (16, 1000, 2048), (17, 100, 31), (33, 257, 4100),
         (65, 2048, 1024), (64, 128, 128), (129, 72, 1000), (128, 256, 64), (300, 1001, 200), (777, 512, 257),
         (1040, 1024, 1024), (4160, 776, 384)]


@pytest.mark.parametrize("M,N,K", SIZES)
@pytest.mark.parametrize("epi,out", [(0, "bf16"), (0, "f16"), (1, "bf16"), (1, "f16"), (2, "f32"), (3, "f32")])
def test_gemm(k, M, N, K, epi, out):
    A, W, rs, cs, bias = operands(M, N, K, M * 7 + N + K + epi)
    if N % 3 == 0:
        bias = None
    # rows padded to whole 16 bytes and to more, and rows that begin anywhere
    first = None
    for pitch, off in ((N, 0), ((N + 15) // 8 * 8, 0), (N + 3, 1)):
        C, full = matrix(M, N, DT[out], pitch, 7, off)
        if epi == 2:
            C.copy_(torch.randn(M, N, device="cuda", generator=gen(N)))
        C0 = C.clone()
        for kernel in KERNELS:
            C.copy_(C0)
            assert k.k_gemm_i8(A, W, rs, cs, bias, C, epi, kernel) is C
            if first is None:
                check_product(C, C0, A, W, rs, cs, bias, epi)
                first = C.clone()
            assert torch.equal(C, first), f"kernel {kernel}, pitch {pitch}"
            assert untouched(C, full, 7, off)
    k.k_i8_check()


# Several tiles of 256 x 256 for each of the pair kernel's CTA pairs (74 on a GPU of 148 SMs): A's blocks kept over a row
# of tiles (K <= 1,024) or both operands streamed, rows of tiles that end inside a pair's share, one tile a row, one row.
PAIR_SIZES = [(9000, 1104, K) for K in (100, 128, 129, 300, 512, 640, 700, 800, 1000, 1024, 1025, 1300, 2048, 4100)] + [
    (8500, 2060, 1000), (40000, 40, 200), (57000, 250, 300), (600, 20000, 130), (250, 60000, 1000), (1, 70000, 1040),
    (33024, 512, 64), (20000, 1001, 1111)]


@pytest.mark.parametrize("M,N,K", PAIR_SIZES)
@pytest.mark.parametrize("epi,out", [(0, "bf16"), (0, "f16"), (1, "bf16"), (1, "f16"), (2, "f32"), (3, "f32")])
def test_gemm_many_tiles_a_pair(k, M, N, K, epi, out):
    A, W, rs, cs, bias = operands(M, N, K, M + N * 3 + K * 5 + epi)
    if K % 2:
        bias = None
    first = None
    for pitch, off in (((N + 7) // 8 * 8, 0), (N + 3, 1)):     # stored by TMA where N suits it, and by the warps
        C, full = matrix(M, N, DT[out], pitch, 7, off)
        if epi == 2:
            C.copy_(torch.randn(M, N, device="cuda", generator=gen(N)))
        C0 = C.clone()
        for kernel in (1, 2, -1, 1):
            C.copy_(C0)
            k.k_gemm_i8(A, W, rs, cs, bias, C, epi, kernel)
            if first is None:
                check_product(C, C0, A, W, rs, cs, bias, epi)
                first = C.clone()
            assert torch.equal(C, first), f"kernel {kernel}, pitch {pitch}"
        assert untouched(C, full, 7, off)
    k.k_i8_check()


@pytest.mark.parametrize("epi,pitch", [(0, 32768), (2, 32768), (3, 32769), (1, 32769)])
def test_pair_offsets_past_32_bits(k, epi, pitch):
    """The pair kernel's rows of A and C more than 2^31 elements into their buffers."""
    M, D, N = 70000, 48, 600
    r = gen(epi)
    q = torch.empty(M, 32768, dtype=torch.int8, device="cuda")[:, 32768 - D:]
    q.copy_(torch.randint(-128, 128, (M, D), device="cuda", generator=r, dtype=torch.int32).to(torch.int8))
    W = torch.randint(-128, 128, (N, D), device="cuda", generator=r, dtype=torch.int32).to(torch.int8)
    rs, cs = torch.rand(M, device="cuda", generator=r) + 0.5, torch.rand(N, device="cuda", generator=r) / 1000
    C = torch.zeros(M, pitch, dtype=torch.float32 if epi >= 2 else torch.bfloat16, device="cuda")[:, :N]
    k.k_gemm_i8(q, W, rs, cs, None, C, epi, 1)
    check_product(C, torch.zeros(M, N, device="cuda"), q, W, rs, cs, None, epi)
    k.k_i8_check()


@pytest.mark.parametrize("M", [1, 20, 300])
def test_gemm_largest_sums(k, M):
    """The longest K at the largest products: the int32 sum comes to 2^31 - 16,384."""
    K = 131071
    A, W, rs, cs, _ = operands(M, 40, K, 5)
    A.fill_(-128)
    W.fill_(-128)
    W[1].fill_(127)
    C = torch.empty(M, 40, device="cuda")
    one = torch.ones(M, device="cuda"), torch.ones(40, device="cuda")
    want = torch.full((M, 40), float(128 * 128 * K), device="cuda")
    want[:, 1] = -128.0 * 127 * K
    for kernel in KERNELS:
        k.k_gemm_i8(A, W, *one, None, C.zero_(), 3, kernel)
        assert torch.equal(C, want), kernel


def test_gemm_nan_scale_marks_its_row(k):
    A, W, rs, cs, bias = operands(70, 96, 64, 3)
    rs[3] = math.nan
    for out, epi in (("bf16", 0), ("f16", 1), ("f32", 2), ("f32", 3)):
        for kernel in KERNELS:
            C = torch.zeros(70, 96, dtype=DT[out], device="cuda")
            k.k_gemm_i8(A, W, rs, cs, bias, C, epi, kernel)
            bad = torch.isnan(C)
            assert bad[3].all() and not bad[[i for i in range(70) if i != 3]].any()


@pytest.mark.parametrize("out", ["bf16", "f16"])
def test_gelu_of_every_size(k, out):
    """The products are zero here, so an output is gelu(bias). It lies between the roundings of the exact value less and
    plus what the GELU before it may be off by: 2.5e-5 of |x| Phi(-|x|) (the polynomial), four roundings of f32, and
    1e-22 below x = -10, where Phi is held."""
    N = 1 << 18
    x = torch.linspace(-12, 12, N, device="cuda")
    A, W = torch.zeros(2, 16, dtype=torch.int8, device="cuda"), torch.zeros(N, 16, dtype=torch.int8, device="cuda")
    d = x.double()
    v = d * torch.special.erfc(-d / math.sqrt(2)) / 2              # erfc keeps the far negative side, ndtr gives 0 there
    e = 2.5e-5 * d.abs() * torch.special.erfc(d.abs() / math.sqrt(2)) / 2 + 4 * U * v.abs() + 1e-22
    C = torch.empty(2, N, dtype=DT[out], device="cuda")
    for kernel in (1, 2):
        k.k_gemm_i8(A, W, torch.ones(2, device="cuda"), torch.ones(N, device="cuda"), x, C, 1, kernel)
        assert (C >= (v - e).to(C.dtype)).all() and (C <= (v + e).to(C.dtype)).all(), kernel


@pytest.mark.parametrize("epi,out", [(1, "bf16"), (2, "f32"), (3, "f32")])
@pytest.mark.parametrize("split", [1, 2, 8])
def test_gemm_gives_up_without_storing(k, split, epi, out):
    """The last CTA of each cluster is given no operands: its waits run out after 2 s, the check says so, and nothing of
    the product is stored. The calls after it are as ever."""
    A, W, rs, cs, bias = operands(19, 300, 2100, 11)
    C, full = matrix(19, 300, DT[out], 304, 7)
    C0 = C.fill_(5).clone()
    k.k_gemm_i8(A, W, rs, cs, bias, C, epi, 64 + 2 + split)
    with pytest.raises(RuntimeError, match="device error"):
        k.k_i8_check()
    assert torch.equal(C, C0) and untouched(C, full, 7)
    k.k_gemm_i8(A, W, rs, cs, bias, C, epi, 2 + split)
    k.k_i8_check()
    check_product(C, C0, A, W, rs, cs, bias, epi)


def test_gemm_offset_vectors(k):
    """Scales and bias that begin on 4 bytes, and operands that are rows of larger matrices."""
    A, W, rs, cs, bias = operands(400, 520, 256, 9)
    want = torch.empty(390, 511, dtype=torch.bfloat16, device="cuda")
    k.k_gemm_i8(A[10:], W[9:], rs[10:].clone(), cs[9:].clone(), bias[9:].clone(), want, 0)
    for kernel in KERNELS:
        got = torch.empty_like(want)
        k.k_gemm_i8(A[10:], W[9:], rs[10:], cs[9:], bias[9:], got, 0, kernel)
        assert torch.equal(got, want), kernel
    check_product(got, None, A[10:], W[9:], rs[10:], cs[9:], bias[9:], 0)


def test_offsets_past_32_bits(k):
    """Rows whose elements lie more than 2^31 elements into their buffers."""
    M, D, pitch = 70000, 48, 32768
    X = torch.empty(M, pitch, dtype=torch.float16, device="cuda")[:, :D]
    X.copy_(torch.randn(M, D, device="cuda", generator=gen(1)))
    q = torch.empty(M, pitch, dtype=torch.int8, device="cuda")[:, :D]
    scale = torch.empty(M, device="cuda")
    k.k_quant_i8(X, q, scale)
    check_codes(q, scale, X.double(), X.double().abs().amax(1) / 127, U)
    W = torch.randint(-127, 128, (40, D), device="cuda", dtype=torch.int32).to(torch.int8)
    cs = torch.full((40,), 0.01, device="cuda")
    for epi, p in ((0, pitch), (2, pitch), (0, pitch + 1)):
        C = torch.zeros(M, p, dtype=torch.float32 if epi else torch.bfloat16, device="cuda")[:, :40]
        k.k_gemm_i8(q, W, scale, cs, None, C, epi)
        check_product(C, torch.zeros(M, 40, device="cuda"), q, W, scale, cs, None, epi)


# ------------------------------------------------------------------------------------------------ together
def block(k, b):
    """A feed-forward block on int8 products: norm with the residual's addition, product + GELU, quantiser, product."""
    k.k_rmsnorm_i8(b["x"], b["delta"], b["g"], b["out"], b["q"], b["s"])
    k.k_gemm_i8(b["q"], b["W1"], b["s"], b["c1"], b["b1"], b["h"], 1)
    k.k_quant_i8(b["h"], b["q2"], b["s2"])
    k.k_gemm_i8(b["q2"], b["W2"], b["s2"], b["c2"], b["b2"], b["out"], 2)


def block_state(k, M, d, ff, seed):
    r = gen(seed)
    e = lambda *n, dtype=torch.float32: torch.empty(*n, dtype=dtype, device="cuda")  # noqa: E731
    b = {"x": torch.randn(M, d, device="cuda", generator=r), "g": 1 + 0.1 * torch.randn(d, device="cuda", generator=r),
         "delta": torch.randn(M, d, device="cuda", generator=r).bfloat16(), "out": e(M, d),
         "q": e(M, d, dtype=torch.int8), "s": e(M), "h": e(M, ff, dtype=torch.bfloat16),
         "q2": e(M, ff, dtype=torch.int8), "s2": e(M), "b1": torch.randn(ff, device="cuda", generator=r) * 0.1,
         "b2": torch.randn(d, device="cuda", generator=r) * 0.1,
         "w1": torch.randn(ff, d, device="cuda", generator=r) / math.sqrt(d),
         "w2": torch.randn(d, ff, device="cuda", generator=r) / math.sqrt(ff)}
    for i, (n, kk) in ((1, (ff, d)), (2, (d, ff))):
        b[f"W{i}"], b[f"c{i}"] = k.k_quant_i8(b[f"w{i}"], e(n, kk, dtype=torch.int8), e(n))
    return b


@pytest.mark.parametrize("M,d,ff", [(1, 256, 1024), (65, 1024, 2048), (520, 1008, 2000), (2080, 1024, 2048)])
def test_block(k, M, d, ff):
    b = block_state(k, M, d, ff, M)
    block(k, b)
    # each step against its definition on what the step before it stored
    s = b["x"] + b["delta"].float()
    t = s.double() * b["g"].double()
    r64 = 1 / torch.sqrt(s.double().square().mean(1) + float(torch.tensor(1e-6)))
    check_codes(b["q"], b["s"], t, t.abs().amax(1) * r64 / 127, ((d / 32 + 10) / 2 + 9) * U)
    check_product(b["h"], None, b["q"], b["W1"], b["s"], b["c1"], b["b1"], 1)
    h = b["h"].double()
    check_codes(b["q2"], b["s2"], h, h.abs().amax(1) / 127, U)
    check_product(b["out"], s, b["q2"], b["W2"], b["s2"], b["c2"], b["b2"], 2)
    # and the whole against the block in 64 bits without quantising: a code is off by up to half a step of a row's
    # largest / 127, uniformly, so by (largest / rms) / (127 sqrt 12) of the row's rms. With a largest of at most 5.5 rms
    # (normal rows of up to 2,048) that is 1.25%; the GELU's rows have a largest of up to 8 rms: 1.8%. Four operands,
    # independent: sqrt(3 * 1.25^2 + 1.8^2) < 2.9%, and GELU passes on at most 1.13 of its input's error: 3.3%
    y = t * r64[:, None]
    f = y @ b["w1"].double().t() + b["b1"].double()
    f = (f * torch.special.ndtr(f)) @ b["w2"].double().t() + b["b2"].double()
    got = b["out"].double() - s.double()
    assert (got - f).norm() <= 0.033 * f.norm()


def test_block_on_another_stream_and_replayed(k):
    """The block on a side stream, two blocks on two streams at once, and two captured graphs replayed on new inputs."""
    M, d, ff = 325, 256, 1024
    blocks = [block_state(k, M, d, ff, 70 + i) for i in range(2)]
    want = []
    for b in blocks:
        block(k, b)
        want.append([b[n].clone() for n in ("out", "q", "q2", "h")])
    torch.cuda.synchronize()
    side = [torch.cuda.Stream() for _ in blocks]
    for _ in range(5):
        for b, s in zip(blocks, side):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                b["out"].zero_()
                block(k, b)
    torch.cuda.synchronize()
    for b, w in zip(blocks, want):
        assert all(torch.equal(b[n], t) for n, t in zip(("out", "q", "q2", "h"), w))
    graphs = []
    for b in blocks:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            block(k, b)
        graphs.append(g)
    blocks[0]["x"].copy_(blocks[1]["x"])
    blocks[0]["delta"].copy_(blocks[1]["delta"])
    for n in ("g", "W1", "c1", "b1", "W2", "c2", "b2"):
        blocks[0][n].copy_(blocks[1][n])
    for _ in range(3):
        for g, s in zip(graphs, side):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for b in blocks:
            assert all(torch.equal(b[n], t) for n, t in zip(("out", "q", "q2", "h"), want[1]))
    del graphs


def test_block_from_threads(k):
    """Four host threads, each with a stream and a block of its own sizes, at the same time: the bits of one after the
    other."""
    import threading
    sizes = [(1, 256, 1024), (325, 512, 1008), (2080, 1024, 2048), (9000, 256, 1104)]
    blocks = [block_state(k, *n, 90 + i) for i, n in enumerate(sizes)]
    names = ("out", "q", "s", "h", "q2", "s2")
    want = []
    for b in blocks:
        block(k, b)
        want.append([b[n].clone() for n in names])
    torch.cuda.synchronize()
    failed = []

    def work(b, w):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(30):
                    for n in names:
                        b[n].zero_()
                    block(k, b)
                    if not all(torch.equal(b[n], t) for n, t in zip(names, w)):
                        failed.append("other bits")
                k.k_i8_check()
        except Exception as e:
            failed.append(repr(e))
    threads = [threading.Thread(target=work, args=a) for a in zip(blocks, want)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed


def test_first_call_of_a_process_captured(k):
    """Each operator's first call of a process inside a stream capture: nothing in it may need an earlier call."""
    import subprocess
    import sys

    from conftest import REPO
    code = """
import torch
from mayfly_chess_b200 import cudanet_py as k
M, K, N = 300, 256, 512
e = lambda *n, dtype=torch.float32: torch.zeros(*n, dtype=dtype, device="cuda")
x, q, s, w, c = torch.ones(M, K, device="cuda"), e(M, K, dtype=torch.int8), e(M), e(N, K, dtype=torch.int8), e(N)
C, B = e(M, N), torch.full((N, K), 2.0, device="cuda")
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    k.k_quant_i8(B, w, c)
    k.k_rmsnorm_i8(x, x, torch.ones_like(c[:K]), x, q, s)
    for kernel in (-1, 1, 10):
        k.k_gemm_i8(q, w, s, c, None, C, 2, kernel)
g.replay()
torch.cuda.synchronize()
k.k_i8_check()
# out = 2 in place, its norm 1, times a weight of 2: K * 2 for each of the three products added
assert (x == 2).all() and ((C / (3 * 2 * K) - 1).abs() < 1e-5).all(), C
"""
    r = subprocess.run([sys.executable, "-c", code], cwd=REPO, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


def test_no_rows(k):
    e = lambda *n, dtype=torch.float32: torch.empty(*n, dtype=dtype, device="cuda")  # noqa: E731
    k.k_quant_i8(e(0, 64), e(0, 64, dtype=torch.int8), e(0))
    k.k_rmsnorm_i8(e(0, 64), e(0, 64), e(64), e(0, 64), e(0, 64, dtype=torch.int8), e(0))
    k.k_gemm_i8(e(0, 64, dtype=torch.int8), torch.ones(8, 64, dtype=torch.int8, device="cuda"), e(0), e(8), None,
                e(0, 8), 3)
    torch.cuda.synchronize()


# ------------------------------------------------------------------------------------------------ refusals
def test_wrapper_refusals(k):
    e = lambda *n, dtype=torch.float32: torch.empty(*n, dtype=dtype, device="cuda")  # noqa: E731
    i8 = torch.int8
    x, q, s, g = e(4, 32), e(4, 32, dtype=i8), e(4), e(32)
    for bad in ((x.double(), q, s), (x.cpu(), q, s), (x, q.cpu(), s), (x, q.float(), s), (x, q[:, :16], s), (x, q, e(5)),
                (x, q, s.half()), (x, q, e(8)[::2]), (x.t(), q, s), (e(32, 4).t(), q, s), (x[0], q[0], s)):
        with pytest.raises(ValueError):
            k.k_quant_i8(*bad)
    for bad in ((x, None, g, x, q, s), (x, x, g, None, q, s), (x, x, g, x.half(), q, s), (x, x[:2], g, x, q, s),
                (x, x, e(31), x, q, s), (x, x.double(), g, x, q, s)):
        with pytest.raises(ValueError):
            k.k_rmsnorm_i8(*bad)
    h = x.half()
    with pytest.raises(RuntimeError, match="delta must be of x's type"):
        k.k_rmsnorm_i8(h, x, g, h, q, s)
    for eps in (0.0, -1e-6, math.nan, math.inf):
        with pytest.raises(RuntimeError, match="eps"):
            k.k_rmsnorm_i8(x, None, g, None, q, s, eps)
    with pytest.raises(RuntimeError, match="32768"):
        k.k_quant_i8(e(1, 32769), e(1, 32769, dtype=i8), e(1))
    A, W, C = e(4, 32, dtype=i8), e(8, 32, dtype=i8), e(4, 8)
    c = e(8)
    for bad in ((A, W[:, :16], s, c, None, C, 3), (A, W, s, c, None, C.t(), 3), (A, W, s, c, None, C, 0),
                (A, W, s, c, None, C.half(), 2), (A.float(), W, s, c, None, C, 3), (A, W, e(3), c, None, C, 3),
                (A, W, s, e(4), None, C, 3), (A, W, s, c, e(7), C, 3), (A, W.cpu(), s, c, None, C, 3)):
        with pytest.raises(ValueError):
            k.k_gemm_i8(*bad)
    with pytest.raises(RuntimeError, match="16"):
        k.k_gemm_i8(e(4, 33, dtype=i8)[:, 1:], W, s, c, None, C, 3)
    with pytest.raises(RuntimeError, match="multiples of 16"):
        k.k_gemm_i8(e(4, 40, dtype=i8)[:, :32], W, s, c, None, C, 3)
    with pytest.raises(RuntimeError, match="epi"):
        k.k_gemm_i8(A, W, s, c, None, C, 4)
    with pytest.raises(RuntimeError, match="kernel"):
        k.k_gemm_i8(A, W, s, c, None, C, 3, 99)
