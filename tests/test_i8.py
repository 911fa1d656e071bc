"""What the int8 entry points refuse on the host, through the C ABI: no GPU, nothing is queued."""
import ctypes

import pytest

P = 1 << 20          # an address that no refused call looks at


@pytest.fixture(scope="module")
def lib():
    from mayfly_chess_b200 import build, cudanet_py
    build.build()
    return cudanet_py.load()


def refused(fn, args, names, reason, **change):
    values = dict(zip(names, args))
    for n in change:
        assert n in values
    values.update(change)
    err = ctypes.create_string_buffer(512)
    assert fn(*values.values(), None, err, 512) == -1
    assert reason in err.value.decode(), err.value


GEMM = ("dtype", "epi", "kernel", "A", "W", "rowscale", "colscale", "bias", "C", "M", "N", "K", "lda", "ldw", "ldc")


@pytest.mark.parametrize("reason,change", [
    ("dtype", {"dtype": 2}), ("dtype", {"dtype": -1}), ("epi", {"epi": 4}), ("epi", {"epi": -1}),
    ("kernel", {"kernel": 77}), ("bad sizes", {"M": -1}), ("bad sizes", {"N": 0}), ("bad sizes", {"K": 0}),
    ("bad sizes", {"K": 131072}), ("bad sizes", {"M": 2 ** 31 - 1}), ("bad sizes", {"N": 2 ** 30 + 1}), ("A is a null", {"A": None}), ("W is a null", {"W": None}),
    ("rowscale is a null", {"rowscale": None}), ("colscale is a null", {"colscale": None}), ("C is a null", {"C": None}),
    ("A is not aligned to 16", {"A": P + 8}), ("W is not aligned to 16", {"W": P + 1}),
    ("rowscale is not aligned to 4", {"rowscale": P + 2}), ("bias is not aligned to 4", {"bias": P + 1}),
    ("C is not aligned to 2", {"C": P + 1}), ("C is not aligned to 4", {"C": P + 2, "epi": 3}),
    ("lda is less", {"lda": 48}), ("ldw is less", {"ldw": 0}), ("ldc is less", {"ldc": 31}),
    ("multiples of 16", {"lda": 72}), ("multiples of 16", {"ldw": 65})])
def test_gemm_refusals(lib, reason, change):
    args = (1, 0, -1, P, P, P, P, P, P, 5, 32, 64, 64, 64, 32)
    refused(lib.cudanet_k_gemm_i8, args, GEMM, reason, **change)


@pytest.mark.parametrize("kernel", [0, 5, 11, 63, 65, 66, 69, 75, 128, -2, 2 ** 31 - 1, -2 ** 31])
def test_gemm_refuses_other_kernels(lib, kernel):
    args = (1, 0, -1, P, P, P, P, P, P, 5, 32, 64, 64, 64, 32)
    refused(lib.cudanet_k_gemm_i8, args, GEMM, "kernel", kernel=kernel)


NORM = ("x_type", "delta_type", "x", "delta", "g", "out", "q", "scale", "M", "D", "ldx", "ldd", "ldo", "ldq", "eps")


@pytest.mark.parametrize("reason,change", [
    ("type", {"x_type": 3}), ("type", {"delta_type": -1}), ("x's type", {"x_type": 1, "delta_type": 0}),
    ("x's type", {"x_type": 0, "delta_type": 2}), ("bad sizes", {"M": -3}), ("bad sizes", {"M": 2 ** 30 + 1}), ("bad sizes", {"D": 0}),
    ("bad sizes", {"D": 32769}), ("eps", {"eps": 0.0}), ("eps", {"eps": float("nan")}), ("eps", {"eps": float("inf")}),
    ("x is a null", {"x": None}), ("g is a null", {"g": None}), ("q is a null", {"q": None}),
    ("scale is a null", {"scale": None}), ("out is a null", {"out": None}), ("out without delta", {"delta": None}),
    ("x is not aligned", {"x": P + 2}), ("delta is not aligned", {"delta": P + 1}), ("out is not aligned", {"out": P + 2}),
    ("ldx is less", {"ldx": 63}), ("ldd is less", {"ldd": 1}), ("ldo is less", {"ldo": -64}), ("ldq is less", {"ldq": 0})])
def test_rmsnorm_refusals(lib, reason, change):
    args = (2, 1, P, P, P, P, P, P, 5, 64, 64, 64, 64, 64, 1e-6)
    refused(lib.cudanet_k_rmsnorm_i8, args, NORM, reason, **change)


QUANT = ("x_type", "x", "q", "scale", "M", "D", "ldx", "ldq")


@pytest.mark.parametrize("reason,change", [
    ("x_type", {"x_type": 3}), ("bad sizes", {"M": -1}), ("bad sizes", {"D": 0}), ("bad sizes", {"D": 32769}),
    ("x is a null", {"x": None}), ("q is a null", {"q": None}), ("scale is a null", {"scale": None}),
    ("x is not aligned", {"x": P + 1}), ("scale is not aligned", {"scale": P + 2}), ("ldx is less", {"ldx": 63}),
    ("ldq is less", {"ldq": 0})])
def test_quant_refusals(lib, reason, change):
    refused(lib.cudanet_k_quant_i8, (0, P, P, P, 5, 64, 64, 64), QUANT, reason, **change)


def test_no_rows_is_nothing_to_do(lib):
    err = ctypes.create_string_buffer(64)
    assert lib.cudanet_k_quant_i8(0, None, None, None, 0, 64, 0, 0, None, err, 64) == 0
    assert lib.cudanet_k_rmsnorm_i8(0, 0, None, None, None, None, None, None, 0, 64, 0, 0, 0, 0, 1e-6, None, err, 64) == 0
    assert lib.cudanet_k_gemm_i8(0, 0, -1, None, None, None, None, None, None, 0, 8, 64, 0, 0, 0, None, err, 64) == 0


def test_wrappers_refuse_host_tensors():
    import torch

    from mayfly_chess_b200 import cudanet_py as k
    x, q, s = torch.ones(2, 16), torch.ones(2, 16, dtype=torch.int8), torch.ones(2)
    with pytest.raises(ValueError, match="CUDA"):
        k.k_quant_i8(x, q, s)
    with pytest.raises(ValueError, match="CUDA"):
        k.k_rmsnorm_i8(x, x, torch.ones(16), x, q, s)
    with pytest.raises(ValueError, match="CUDA"):
        k.k_gemm_i8(q, q, s, s, None, torch.empty(2, 2), 3)


class Fake:
    """What the wrappers ask of a tensor on device 0, without its memory."""

    def __init__(self, dtype, *shape):
        import torch
        self.dtype, self.shape, self.device = dtype, torch.Size(shape), "cuda:0"

    def stride(self, i=None):
        st = [1]
        for n in self.shape[:0:-1]:
            st.insert(0, st[0] * n)
        return tuple(st) if i is None else st[i]

    def get_device(self):
        return 0

    def is_contiguous(self):
        return True

    def data_ptr(self):
        return P


@pytest.fixture
def calls(monkeypatch):
    """The wrappers with a library that notes its calls in place of the real one."""
    from mayfly_chess_b200 import cudanet_py as k
    seen = []

    class Lib:
        def __getattr__(self, name):
            return lambda *args: seen.append((name, args)) or 0
    once = k._I8Once()
    once.device, once.stream, once.lib = (lambda: 0), (lambda dev: 0), Lib()
    monkeypatch.setattr(k, "_i8_once", once)
    return k, seen


BIG = 2 ** 32 + 32   # its low 32 bits are a size like any other


@pytest.mark.parametrize("M,D", [(BIG, 64), (4, BIG), (2 ** 31, 64), (BIG, BIG)])
def test_wrappers_refuse_rows_over_32_bits(calls, M, D):
    import torch
    k, seen = calls
    f32 = torch.float32
    x, q, g, s = Fake(f32, M, D), Fake(torch.int8, M, D), Fake(f32, D), Fake(f32, M)
    with pytest.raises(ValueError, match="32 bits"):
        k.k_quant_i8(x, q, s)
    with pytest.raises(ValueError, match="32 bits"):
        k.k_rmsnorm_i8(x, x, g, x, q, s)
    assert not seen


@pytest.mark.parametrize("change", [{"M": BIG}, {"N": BIG}, {"K": BIG}, {"epi": 2 ** 32 + 2}, {"kernel": 2 ** 32 + 1},
                                    {"kernel": 2 ** 32 - 1}, {"epi": 2 ** 31, "kernel": -2 ** 31 - 1}])
def test_gemm_wrapper_refuses_numbers_over_32_bits(calls, change):
    import torch
    k, seen = calls
    v = {"M": 4, "N": 32, "K": 64, "epi": 3, "kernel": -1, **change}
    i8, f32 = torch.int8, torch.float32
    with pytest.raises(ValueError, match="32 bits"):
        k.k_gemm_i8(Fake(i8, v["M"], v["K"]), Fake(i8, v["N"], v["K"]), Fake(f32, v["M"]), Fake(f32, v["N"]), None,
                    Fake(f32, v["M"], v["N"]), v["epi"], v["kernel"])
    assert not seen


def test_wrappers_pass_what_they_are_given(calls):
    """The same stand-ins with sizes in range reach the library, so the refusals above are of the sizes."""
    import torch
    k, seen = calls
    i8, f32 = torch.int8, torch.float32
    x, q, g, s = Fake(f32, 5, 64), Fake(i8, 5, 64), Fake(f32, 64), Fake(f32, 5)
    k.k_quant_i8(x, q, s)
    k.k_rmsnorm_i8(x, x, g, x, q, s)
    k.k_gemm_i8(q, Fake(i8, 32, 64), s, Fake(f32, 32), None, Fake(f32, 5, 32), 3, 10)
    k.k_gemm_i8(q, Fake(i8, 32, 64), s, Fake(f32, 32), None, Fake(f32, 5, 32), 4, -2)     # the library's to refuse
    assert [n for n, _ in seen] == ["cudanet_k_quant_i8", "cudanet_k_rmsnorm_i8"] + ["cudanet_k_gemm_i8"] * 2
    assert seen[2][1][9:12] == (5, 32, 64) and seen[3][1][1:3] == (4, -2)


def test_check_asks_the_streams_device(monkeypatch):
    """The library reads the word of the current device, so the stream's has to be it while the library is called."""
    import contextlib

    import torch
    from mayfly_chess_b200 import cudanet_py as k
    current, seen = [0], []

    @contextlib.contextmanager
    def device(d):
        before, current[0] = current[0], torch.device(d).index
        yield
        current[0] = before

    class Stream:
        device, cuda_stream = torch.device("cuda:3"), 77

    class Lib:
        def cudanet_k_i8_check(self, stream, err, err_len):
            seen.append((current[0], stream.value))
            return -1 if len(seen) > 1 else 0
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(k, "load", lambda dll=None: Lib())
    k.k_i8_check(Stream())
    with pytest.raises(RuntimeError):
        k.k_i8_check(Stream())
    assert seen == [(3, 77)] * 2 and current[0] == 0
