"""libcudanet_b200.so from Python through ctypes: the reference backend's Python interface, unchanged.

    net = CudaNet("net.cnw")
    pol, val, qv = net.evaluate(ids, cast, hm, ep, I, M)

This mirrors mayfly/chess/cudanet/cudanet_py.py:87-178 (class CudaNet): the same constructor
(weights_path, device=0, dll=None), the same evaluate(ids, cast, hm, ep, I, M) -> (pol, val, qv) with the same
shape and dtype checks (bool M is taken too), fingerprint(), profile(B, reps), close() and the context
manager, the same exceptions (ValueError for bad shapes or batch sizes, RuntimeError with the library's reason
for a failed call). The inputs are what MCTS._prepare builds: ids (B, 64) int64, cast (B, 4) float32, hm (B,)
int64, ep (B,) int64, I (B, wide) int64 and M (B, wide) uint8. The outputs are float32 pol (B, wide) (raw policy
logits at each row's legal moves, 0 on padding), val (B,) and qv (B, wide).

Additions: evaluate_logits (also the full (B, 8324) logits), begin/end (two batches in flight),
evaluate_device (torch CUDA tensors in and out, queued on a stream), precision, check, calibrate (the input
ranges an e4m3 weight file's static scales come from), k_* single-kernel entry points for unit tests, and the int8
linear layer with dynamic scales (k_rmsnorm_i8, k_quant_i8, k_gemm_i8, k_i8_check; asynchronous on the current stream).

The library is MAYFLY_CUDANET_DLL, else libcudanet_b200.so beside this file. There is no fallback: if the
library is missing the constructor raises.
"""
import ctypes
import os
import threading

import numpy as np

HERE = os.path.dirname(os.path.abspath(__file__))
MAX_BATCH = 1024        # the library's default (env MAYFLY_CUDANET_MAX_BATCH when a net is made)
MAX_WIDE = 256
N_MOVES = 4162
ERR_LEN = 2048

_libs = {}
_load_lock = threading.Lock()


def dll_path(dll=None):
    """Which library file a handle binds: the explicit argument, then $MAYFLY_CUDANET_DLL, then the build in this
    package's folder."""
    for choice in (dll, os.environ.get("MAYFLY_CUDANET_DLL")):
        if choice:
            return choice
    return os.path.join(HERE, "libcudanet_b200.so")


def load(dll=None):
    """The library, loaded once per path, with every entry point's signature declared."""
    path = os.path.abspath(dll_path(dll))
    with _load_lock:
        if path in _libs:
            return _libs[path]
        if not os.path.exists(path):
            raise FileNotFoundError(f"no libcudanet_b200.so at {path} (build it: python -m mayfly_chess_b200.build)")
        lib = ctypes.CDLL(path)
        vp, i32, cp = ctypes.c_void_p, ctypes.c_int, ctypes.c_char_p
        lib.cudanet_create.argtypes = [cp, i32, cp, i32]
        lib.cudanet_create.restype = vp
        lib.cudanet_evaluate.argtypes = [vp, i32, i32] + [vp] * 9 + [cp, i32]
        lib.cudanet_evaluate.restype = i32
        lib.cudanet_evaluate_logits.argtypes = [vp, i32, i32] + [vp] * 10 + [cp, i32]
        lib.cudanet_evaluate_logits.restype = i32
        lib.cudanet_begin.argtypes = [vp, i32, i32] + [vp] * 6 + [cp, i32]
        lib.cudanet_begin.restype = i32
        lib.cudanet_end.argtypes = [vp, vp, vp, vp, cp, i32]
        lib.cudanet_end.restype = i32
        lib.cudanet_fingerprint.argtypes = [vp, cp, i32]
        lib.cudanet_fingerprint.restype = i32
        lib.cudanet_precision.argtypes = [vp, cp, i32]
        lib.cudanet_precision.restype = i32
        lib.cudanet_max_batch.argtypes = [vp]
        lib.cudanet_max_batch.restype = i32
        lib.cudanet_profile.argtypes = [vp, i32, i32, ctypes.POINTER(ctypes.c_double), i32, cp, i32]
        lib.cudanet_profile.restype = i32
        lib.cudanet_profile_names.argtypes = [cp, i32]
        lib.cudanet_profile_names.restype = i32
        lib.cudanet_destroy.argtypes = [vp]
        lib.cudanet_destroy.restype = None
        lib.cudanet_evaluate_device.argtypes = [vp, i32, i32] + [vp] * 10 + [cp, i32]
        lib.cudanet_evaluate_device.restype = i32
        lib.cudanet_check.argtypes = [vp, vp, cp, i32]
        lib.cudanet_check.restype = i32
        lib.cudanet_k_gemm.argtypes = [i32, i32, i32, vp, vp, vp, vp, i32, i32, i32, i32, vp, cp, i32]
        lib.cudanet_k_gemm.restype = i32
        lib.cudanet_k_gemm_noalloc.argtypes = [i32, i32, i32, vp, vp, vp, vp, i32, i32, i32, i32, vp, cp, i32]
        lib.cudanet_k_gemm_noalloc.restype = i32
        lib.cudanet_k_gemm_resln.argtypes = [i32, vp, vp, vp, vp, vp, vp, vp, i32, i32, i32, vp, cp, i32]
        lib.cudanet_k_gemm_resln.restype = i32
        lib.cudanet_k_attention.argtypes = [i32, vp, vp, i32, i32, i32, vp, cp, i32]
        lib.cudanet_k_attention.restype = i32
        lib.cudanet_k_attention_tc.argtypes = [i32, vp, vp, i32, i32, i32, vp, cp, i32]
        lib.cudanet_k_attention_tc.restype = i32
        lib.cudanet_k_attention_kernel.argtypes = [i32, i32, i32, vp, vp, i32, i32, i32, ctypes.c_float, vp, cp, i32]
        lib.cudanet_k_attention_kernel.restype = i32
        lib.cudanet_k_attention_cls.argtypes = [i32, vp, vp, i32, i32, i32, vp, cp, i32]
        lib.cudanet_k_attention_cls.restype = i32
        lib.cudanet_k_layernorm.argtypes = [i32, vp, vp, vp, vp, i32, i32, i32, vp, cp, i32]
        lib.cudanet_k_layernorm.restype = i32
        f32 = ctypes.c_float
        lib.cudanet_calibrate.argtypes = [vp, i32, vp, vp, vp, vp, vp, i32, cp, i32]
        lib.cudanet_calibrate.restype = i32
        lib.cudanet_k_gemm_f8.argtypes = [i32, i32, vp, vp, vp, vp, f32, vp, i32, i32, i32, i32, vp, cp, i32]
        lib.cudanet_k_gemm_f8.restype = i32
        lib.cudanet_k_attention_f8.argtypes = [vp, vp, i32, i32, i32, f32, vp, cp, i32]
        lib.cudanet_k_attention_f8.restype = i32
        lib.cudanet_k_layernorm_f8.argtypes = [i32, vp, vp, vp, vp, i32, i32, i32, f32, vp, cp, i32]
        lib.cudanet_k_layernorm_f8.restype = i32
        lib.cudanet_evaluate_keys.argtypes = [vp, i32, i32] + [vp] * 8 + [cp, i32]
        lib.cudanet_evaluate_keys.restype = i32
        lib.cudanet_begin_keys.argtypes = [vp, i32, i32] + [vp] * 5 + [cp, i32]
        lib.cudanet_begin_keys.restype = i32
        lib.cudanet_encode_keys.argtypes = [vp, vp, vp, i32, vp, vp, vp, vp, vp, cp, i32]
        lib.cudanet_encode_keys.restype = i32
        i64 = ctypes.c_int64
        lib.cudanet_k_rmsnorm_i8.argtypes = [i32, i32, vp, vp, vp, vp, vp, vp, i32, i32, i64, i64, i64, i64, f32, vp,
                                             cp, i32]
        lib.cudanet_k_rmsnorm_i8.restype = i32
        lib.cudanet_k_quant_i8.argtypes = [i32, vp, vp, vp, i32, i32, i64, i64, vp, cp, i32]
        lib.cudanet_k_quant_i8.restype = i32
        lib.cudanet_k_gemm_i8.argtypes = [i32, i32, i32, vp, vp, vp, vp, vp, vp, i32, i32, i32, i64, i64, i64, vp, cp,
                                          i32]
        lib.cudanet_k_gemm_i8.restype = i32
        lib.cudanet_k_i8_check.argtypes = [vp, cp, i32]
        lib.cudanet_k_i8_check.restype = i32
        _libs[path] = lib
        return lib


def _as_c(value, dtype, shape, name):
    """`value` as a C-ordered array of `dtype` that the library can read in place; numpy makes a new array only
    when the dtype or the memory order has to change (a bool mask is reinterpreted as bytes, never copied).
    ValueError names the argument when its shape is not `shape`."""
    arr = np.asarray(value)
    if arr.dtype == np.bool_ and dtype is np.uint8:
        arr = arr.view(np.uint8)
    arr = np.require(np.atleast_1d(arr), dtype=dtype, requirements="C")
    if arr.shape == shape:
        return arr
    raise ValueError(f"{name}: shape {arr.shape}, expected {shape}")


# The six position inputs MCTS._prepare hands the evaluator: name, element type and shape for (B, wide).
_POSITION_INPUTS = (("ids", np.int64, lambda B, w: (B, 64)), ("cast", np.float32, lambda B, w: (B, 4)),
                    ("hm", np.int64, lambda B, w: (B,)), ("ep", np.int64, lambda B, w: (B,)),
                    ("I", np.int64, lambda B, w: (B, w)), ("M", np.uint8, lambda B, w: (B, w)))
# The key-fed form: transposition keys instead of the encoded board.
_KEY_INPUTS = (("keys", np.uint64, lambda B, w: (B, 10)), ("ep_sq", np.int64, lambda B, w: (B,)),
               ("clock", np.int64, lambda B, w: (B,)), ("I", np.int64, lambda B, w: (B, w)),
               ("M", np.uint8, lambda B, w: (B, w)))


def _p(a):
    return a.ctypes.data_as(ctypes.c_void_p)


def _msg(err):
    return err.value.decode("utf-8", "replace")


class CudaNet:
    """One evaluator handle: the weights on one B200, a CUDA graph per batch size. One call at a time."""

    def __init__(self, weights_path, device=0, dll=None):
        self.path, self.device, self.dll = os.path.abspath(weights_path), int(device), dll_path(dll)
        self._lib, self._lock, self._h = load(self.dll), threading.Lock(), None
        reason = ctypes.create_string_buffer(ERR_LEN)
        handle = self._lib.cudanet_create(self.path.encode("utf-8"), self.device, reason, ERR_LEN)
        if handle:
            self._h = ctypes.c_void_p(handle)
            self.max_batch = int(self._lib.cudanet_max_batch(self._h))
            return
        raise RuntimeError(f"cudanet_create({self.path}): {_msg(reason)}")

    def _batch_dims(self, I):
        """(B, wide) of a call, from the move-index matrix I, after the checks every entry point makes."""
        if self._h is None:
            raise RuntimeError("CudaNet is closed")
        shape = np.shape(I)
        if len(shape) != 2:
            raise ValueError(f"I: shape {shape}, expected (B, wide)")
        B, wide = shape
        if B < 1 or B > self.max_batch:
            raise ValueError(f"batch {B}: cudanet takes 1 to {self.max_batch} (env MAYFLY_CUDANET_MAX_BATCH)")
        if wide < 1:
            raise ValueError("wide must be at least 1")
        return B, wide

    def _convert(self, spec, values):
        B, wide = self._batch_dims(values[-2])
        return (B, wide) + tuple(_as_c(v, dt, shape(B, wide), name) for (name, dt, shape), v in zip(spec, values))

    def _inputs(self, ids, cast, hm, ep, I, M):
        return self._convert(_POSITION_INPUTS, (ids, cast, hm, ep, I, M))

    def evaluate(self, ids, cast, hm, ep, I, M):
        """One batch. Returns (pol (B, wide), val (B,), qv (B, wide)) float32."""
        B, wide, ids, cast, hm, ep, I, M = self._inputs(ids, cast, hm, ep, I, M)
        pol = np.zeros((B, wide), np.float32)
        val = np.zeros(B, np.float32)
        qv = np.zeros((B, wide), np.float32)
        err = ctypes.create_string_buffer(ERR_LEN)
        with self._lock:
            rc = self._lib.cudanet_evaluate(self._h, B, wide, _p(ids), _p(cast), _p(hm), _p(ep), _p(I), _p(M),
                                            _p(pol), _p(val), _p(qv), err, ERR_LEN)
        if rc != 0:
            raise RuntimeError(f"cudanet_evaluate: {_msg(err)}")
        return pol, val, qv

    def _key_inputs(self, keys, ep_sq, clock, I, M):
        return self._convert(_KEY_INPUTS, (keys, ep_sq, clock, I, M))

    def evaluate_keys(self, keys, ep_sq, clock, I, M):
        """evaluate from transposition keys: keys (B, 10) uint64 = Board._transposition_key()[0:10] (turn and
        castling rights as integers), ep_sq (B,) the key's en passant square or -1 for None, clock (B,) the
        halfmove clocks. The GPU encodes them exactly as mayfly/chess/encode.py encode_keys does."""
        B, wide, keys, ep_sq, clock, I, M = self._key_inputs(keys, ep_sq, clock, I, M)
        pol = np.zeros((B, wide), np.float32)
        val = np.zeros(B, np.float32)
        qv = np.zeros((B, wide), np.float32)
        err = ctypes.create_string_buffer(ERR_LEN)
        with self._lock:
            rc = self._lib.cudanet_evaluate_keys(self._h, B, wide, _p(keys), _p(ep_sq), _p(clock), _p(I), _p(M),
                                                 _p(pol), _p(val), _p(qv), err, ERR_LEN)
        if rc != 0:
            raise RuntimeError(f"cudanet_evaluate_keys: {_msg(err)}")
        return pol, val, qv

    def begin_keys(self, keys, ep_sq, clock, I, M):
        """begin from transposition keys (see evaluate_keys); end() returns the outputs."""
        B, wide, keys, ep_sq, clock, I, M = self._key_inputs(keys, ep_sq, clock, I, M)
        err = ctypes.create_string_buffer(ERR_LEN)
        with self._lock:
            rc = self._lib.cudanet_begin_keys(self._h, B, wide, _p(keys), _p(ep_sq), _p(clock), _p(I), _p(M), err,
                                              ERR_LEN)
            if rc == 0:
                self._fly = getattr(self, "_fly", []) + [(B, wide)]
        if rc != 0:
            raise RuntimeError(f"cudanet_begin_keys: {_msg(err)}")

    def evaluate_logits(self, ids, cast, hm, ep, I, M):
        """evaluate, plus the full logits (B, 2 * 4162) float32: policy, then qvalue."""
        B, wide, ids, cast, hm, ep, I, M = self._inputs(ids, cast, hm, ep, I, M)
        pol = np.zeros((B, wide), np.float32)
        val = np.zeros(B, np.float32)
        qv = np.zeros((B, wide), np.float32)
        logits = np.zeros((B, 2 * N_MOVES), np.float32)
        err = ctypes.create_string_buffer(ERR_LEN)
        with self._lock:
            rc = self._lib.cudanet_evaluate_logits(self._h, B, wide, _p(ids), _p(cast), _p(hm), _p(ep), _p(I),
                                                   _p(M), _p(pol), _p(val), _p(qv), _p(logits), err, ERR_LEN)
        if rc != 0:
            raise RuntimeError(f"cudanet_evaluate_logits: {_msg(err)}")
        return pol, val, qv, logits

    def begin(self, ids, cast, hm, ep, I, M):
        """Queue one batch (at most two in flight); end() returns the oldest one's outputs."""
        B, wide, ids, cast, hm, ep, I, M = self._inputs(ids, cast, hm, ep, I, M)
        err = ctypes.create_string_buffer(ERR_LEN)
        with self._lock:
            rc = self._lib.cudanet_begin(self._h, B, wide, _p(ids), _p(cast), _p(hm), _p(ep), _p(I), _p(M), err,
                                         ERR_LEN)
            if rc == 0:
                self._fly = getattr(self, "_fly", []) + [(B, wide)]
        if rc != 0:
            raise RuntimeError(f"cudanet_begin: {_msg(err)}")

    def end(self):
        fly = getattr(self, "_fly", [])
        if not fly:
            raise RuntimeError("cudanet_end: no batch in flight")
        B, wide = fly[0]
        pol = np.zeros((B, wide), np.float32)
        val = np.zeros(B, np.float32)
        qv = np.zeros((B, wide), np.float32)
        err = ctypes.create_string_buffer(ERR_LEN)
        with self._lock:
            self._fly = fly[1:]
            rc = self._lib.cudanet_end(self._h, _p(pol), _p(val), _p(qv), err, ERR_LEN)
        if rc != 0:
            raise RuntimeError(f"cudanet_end: {_msg(err)}")
        return pol, val, qv

    def evaluate_device(self, ids, cast, hm, ep, I, M, pol, val, qv, stream=None):
        """One batch on torch CUDA tensors of the handle's device (outputs preallocated float32), queued on
        `stream` (a torch.cuda.Stream, default the current stream) without waiting."""
        import torch
        if self._h is None:
            raise RuntimeError("CudaNet is closed")
        B, wide = I.shape
        for name, t, dt in (("ids", ids, torch.int64), ("cast", cast, torch.float32), ("hm", hm, torch.int64),
                            ("ep", ep, torch.int64), ("I", I, torch.int64), ("M", M, torch.uint8),
                            ("pol", pol, torch.float32), ("val", val, torch.float32), ("qv", qv, torch.float32)):
            if not t.is_cuda or t.dtype != dt or not t.is_contiguous():
                raise ValueError(f"{name}: needs a contiguous CUDA {dt} tensor")
        s = stream if stream is not None else torch.cuda.current_stream()
        err = ctypes.create_string_buffer(ERR_LEN)
        with self._lock:
            rc = self._lib.cudanet_evaluate_device(self._h, B, wide, ids.data_ptr(), cast.data_ptr(),
                                                   hm.data_ptr(), ep.data_ptr(), I.data_ptr(), M.data_ptr(),
                                                   pol.data_ptr(), val.data_ptr(), qv.data_ptr(),
                                                   ctypes.c_void_p(s.cuda_stream), err, ERR_LEN)
        if rc != 0:
            raise RuntimeError(f"cudanet_evaluate_device: {_msg(err)}")

    def check(self, stream=None):
        """Wait for the handle's work (and `stream`) and raise if a device-side wait failed."""
        err = ctypes.create_string_buffer(ERR_LEN)
        sp = ctypes.c_void_p(stream.cuda_stream) if stream is not None else None
        with self._lock:
            rc = self._lib.cudanet_check(self._h, sp, err, ERR_LEN)
        if rc != 0:
            raise RuntimeError(f"cudanet_check: {_msg(err)}")

    def fingerprint(self):
        """The weight file's fingerprint, as mcts_cpp.fingerprint computes it for the checkpoint."""
        if self._h is None:
            raise RuntimeError("CudaNet is closed")
        buf = ctypes.create_string_buffer(256)
        if self._lib.cudanet_fingerprint(self._h, buf, len(buf)) < 0:
            raise RuntimeError("cudanet_fingerprint failed")
        return buf.value.decode("utf-8", "replace")

    def calibrate(self, ids, cast, hm, ep):
        """Runs the handle's 16-bit pass on these positions and returns max |.| of each layer's four product
        inputs (qkv, out, ff1, ff2) as float32 (layers, 4)."""
        if self._h is None:
            raise RuntimeError("CudaNet is closed")
        B, _ = self._batch_dims(np.empty((np.shape(ids)[0], 1)))
        ids, cast, hm, ep = (_as_c(v, dt, shape(B, 1), name)
                             for (name, dt, shape), v in zip(_POSITION_INPUTS[:4], (ids, cast, hm, ep)))
        out = np.zeros(4 * 256, np.float32)
        err = ctypes.create_string_buffer(ERR_LEN)
        with self._lock:
            k = self._lib.cudanet_calibrate(self._h, B, _p(ids), _p(cast), _p(hm), _p(ep), _p(out), out.size, err,
                                            ERR_LEN)
        if k < 0:
            raise RuntimeError(f"cudanet_calibrate: {_msg(err)}")
        return out[:k].reshape(-1, 4).copy()

    def precision(self):
        buf = ctypes.create_string_buffer(32)
        if self._lib.cudanet_precision(self._h, buf, len(buf)) < 0:
            raise RuntimeError("cudanet_precision failed")
        return buf.value.decode()

    def profile(self, B, reps=20):
        """Milliseconds a pass by step at batch B (an empty board, eager, an event after each step), the mean of
        reps passes, and last graph_pass, the whole pass as a CUDA graph. A dict in pass order."""
        if self._h is None:
            raise RuntimeError("CudaNet is closed")
        buf = ctypes.create_string_buffer(512)
        self._lib.cudanet_profile_names(buf, len(buf))
        names = buf.value.decode("utf-8").split(",")
        ms = (ctypes.c_double * len(names))()
        err = ctypes.create_string_buffer(ERR_LEN)
        with self._lock:
            k = self._lib.cudanet_profile(self._h, int(B), int(reps), ms, len(names), err, ERR_LEN)
        if k < 0:
            raise RuntimeError(f"cudanet_profile: {_msg(err)}")
        return dict(zip(names[:k], list(ms)[:k]))

    def close(self):
        if getattr(self, "_h", None) is not None:
            self._lib.cudanet_destroy(self._h)
            self._h = None

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


# ------------------------------------------------------------------------------------------------ kernels
def _dtype_code(t):
    import torch
    if t.dtype == torch.float16:
        return 0
    if t.dtype == torch.bfloat16:
        return 1
    raise ValueError(f"16-bit float tensors only, got {t.dtype}")


def _stream():
    import torch
    return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


def encode_keys_device(keys, ep_sq, clock, dll=None):
    """The GPU batch encoder on torch CUDA tensors: keys (B, 10) int64/uint64 words, ep_sq (B,) int64 (-1 for
    None), clock (B,) int64, on the current stream. Returns (ids (B, 64) int64, cast (B, 4) float32, hm (B,)
    int64, ep (B,) int64), encode.py encode_keys' values."""
    import torch
    lib = load(dll)
    B = keys.shape[0]
    for name, t in (("keys", keys), ("ep_sq", ep_sq), ("clock", clock)):
        if not t.is_cuda or t.element_size() != 8 or not t.is_contiguous():
            raise ValueError(f"{name}: needs a contiguous CUDA tensor of 64-bit words")
    if tuple(keys.shape) != (B, 10) or tuple(ep_sq.shape) != (B,) or tuple(clock.shape) != (B,):
        raise ValueError("keys (B, 10), ep_sq (B,), clock (B,)")
    dev = keys.device
    ids = torch.empty(B, 64, dtype=torch.int64, device=dev)
    cast = torch.empty(B, 4, dtype=torch.float32, device=dev)
    hm = torch.empty(B, dtype=torch.int64, device=dev)
    ep = torch.empty(B, dtype=torch.int64, device=dev)
    err = ctypes.create_string_buffer(ERR_LEN)
    rc = lib.cudanet_encode_keys(keys.data_ptr(), ep_sq.data_ptr(), clock.data_ptr(), B, ids.data_ptr(),
                                 cast.data_ptr(), hm.data_ptr(), ep.data_ptr(), _stream(), err, ERR_LEN)
    if rc != 0:
        raise RuntimeError(f"cudanet_encode_keys: {_msg(err)}")
    return ids, cast, hm, ep


def keys_from_tuples(keys):
    """Board._transposition_key() tuples (pawns .. castling rights, en passant square or None) as the arrays
    the key entry points take: (keys (B, 10) uint64, ep_sq (B,) int64 with -1 for None)."""
    B = len(keys)
    K = np.array([[int(k[j]) for j in range(10)] for k in keys], dtype=np.uint64).reshape(B, 10)
    ep = np.array([-1 if k[10] is None else int(k[10]) for k in keys], dtype=np.int64)
    return K, ep


def encode_keys(keys, hms, device=0, dll=None):
    """mayfly/chess/encode.py:73-100 encode_keys(keys, hms) with the same arguments and results (numpy ids
    (B, 64) int64, cast (B, 4) float32, hm (B,) int64, ep (B,) int64), computed by the GPU encoder."""
    import torch
    K, ep_sq = keys_from_tuples(keys)
    clock = np.asarray(hms, np.int64).reshape(len(keys))
    with torch.cuda.device(device):
        t = [torch.from_numpy(a.view(np.int64) if a.dtype == np.uint64 else a).cuda() for a in (K, ep_sq, clock)]
        out = encode_keys_device(*t, dll=dll)
        torch.cuda.current_stream().synchronize()
    return tuple(o.cpu().numpy() for o in out)


def k_gemm(A, W, bias, C, epi, bn=0, dll=None):
    """C = A W^T + epilogue on the tensor cores (epi 0 bias, 1 bias+GELU, 2 C += (f32), 3 f32 out)."""
    lib = load(dll)
    M, K = A.shape
    N = W.shape[0]
    err = ctypes.create_string_buffer(ERR_LEN)
    rc = lib.cudanet_k_gemm(_dtype_code(A), int(epi), int(bn), A.data_ptr(), W.data_ptr(), bias.data_ptr(),
                            C.data_ptr(), M, N, K, C.stride(0), _stream(), err, ERR_LEN)
    if rc != 0:
        raise RuntimeError(f"cudanet_k_gemm: {_msg(err)}")
    return C


def k_gemm_noalloc(A, W, bias, C, epi, bn=0, dll=None):
    """k_gemm without any device allocation: for callers that cannot call cudaMalloc (their GPU memory is
    reserved up front, or they must not stall in-flight work on an allocation). Its scratch is a static device
    array shared by every call; calls that overlap on the GPU race on it."""
    lib = load(dll)
    M, K = A.shape
    N = W.shape[0]
    err = ctypes.create_string_buffer(ERR_LEN)
    rc = lib.cudanet_k_gemm_noalloc(_dtype_code(A), int(epi), int(bn), A.data_ptr(), W.data_ptr(), bias.data_ptr(),
                                    C.data_ptr(), M, N, K, C.stride(0), _stream(), err, ERR_LEN)
    if rc != 0:
        raise RuntimeError(f"cudanet_k_gemm_noalloc: {_msg(err)}")
    return C


def k_gemm_resln(A, W, bias, X, g, b, H, dll=None):
    """X += A W^T + bias (f32, in place), then H = LayerNorm(X) * g + b (16-bit), in one fused kernel."""
    lib = load(dll)
    M, K = A.shape
    N = W.shape[0]
    err = ctypes.create_string_buffer(ERR_LEN)
    rc = lib.cudanet_k_gemm_resln(_dtype_code(A), A.data_ptr(), W.data_ptr(), bias.data_ptr(), X.data_ptr(),
                                  g.data_ptr(), b.data_ptr(), H.data_ptr(), M, N, K, _stream(), err, ERR_LEN)
    if rc != 0:
        raise RuntimeError(f"cudanet_k_gemm_resln: {_msg(err)}")
    return X, H


def k_attention(qkv, att, B, d, heads, dll=None):
    lib = load(dll)
    err = ctypes.create_string_buffer(ERR_LEN)
    rc = lib.cudanet_k_attention(_dtype_code(qkv), qkv.data_ptr(), att.data_ptr(), B, d, heads, _stream(), err,
                                 ERR_LEN)
    if rc != 0:
        raise RuntimeError(f"cudanet_k_attention: {_msg(err)}")
    return att


def k_attention_kernel(qkv, att, B, d, heads, kernel, mul=1.0, dll=None):
    """One attention launch on a chosen kernel (0 mma.sync, 1 two-group, 4 four-group tensor-memory, -1 the
    evaluator's choice); att uint8 gets e4m3 of att * mul (bf16 qkv), else att in qkv's type."""
    import torch
    lib = load(dll)
    err = ctypes.create_string_buffer(ERR_LEN)
    rc = lib.cudanet_k_attention_kernel(_dtype_code(qkv), 1 if att.dtype == torch.uint8 else 0, int(kernel),
                                        qkv.data_ptr(), att.data_ptr(), B, d, heads, float(mul), _stream(), err,
                                        ERR_LEN)
    if rc != 0:
        raise RuntimeError(f"cudanet_k_attention_kernel: {_msg(err)}")
    return att


def k_attention_tc(qkv, att, B, d, heads, dll=None):
    """k_attention on the tensor-memory (tcgen05) kernel, head width 64."""
    lib = load(dll)
    err = ctypes.create_string_buffer(ERR_LEN)
    rc = lib.cudanet_k_attention_tc(_dtype_code(qkv), qkv.data_ptr(), att.data_ptr(), B, d, heads, _stream(), err,
                                    ERR_LEN)
    if rc != 0:
        raise RuntimeError(f"cudanet_k_attention_tc: {_msg(err)}")
    return att


def k_attention_cls(qkv, att, B, d, heads, dll=None):
    """att [B, d] = attention of each board's CLS query (token 0) over its 65 tokens."""
    lib = load(dll)
    err = ctypes.create_string_buffer(ERR_LEN)
    rc = lib.cudanet_k_attention_cls(_dtype_code(qkv), qkv.data_ptr(), att.data_ptr(), B, d, heads, _stream(), err,
                                     ERR_LEN)
    if rc != 0:
        raise RuntimeError(f"cudanet_k_attention_cls: {_msg(err)}")
    return att


def k_layernorm(x, g, b, h, n, d, row_stride=1, dll=None):
    lib = load(dll)
    err = ctypes.create_string_buffer(ERR_LEN)
    rc = lib.cudanet_k_layernorm(_dtype_code(h), x.data_ptr(), g.data_ptr(), b.data_ptr(), h.data_ptr(), n, d,
                                 row_stride, _stream(), err, ERR_LEN)
    if rc != 0:
        raise RuntimeError(f"cudanet_k_layernorm: {_msg(err)}")
    return h


# ------------------------------------------------------------------------------------------------ FP8 kernels
def _e4m3(t, name):
    import torch
    if t.dtype not in (torch.float8_e4m3fn, torch.uint8):
        raise ValueError(f"{name}: e4m3 bytes (torch.float8_e4m3fn or uint8) only, got {t.dtype}")


def k_gemm_f8(A, W, colscale, bias, C, epi, out_scale_inv=1.0, bn=0, dll=None):
    """C = epilogue(A W^T * colscale + bias) with e4m3 A and W (epi 0 bf16 out, 2 C += (f32), 3 f32 out,
    4 e4m3 out of gelu(.) * out_scale_inv, 5 C += (bf16))."""
    _e4m3(A, "A")
    _e4m3(W, "W")
    lib = load(dll)
    M, K = A.shape
    N = W.shape[0]
    err = ctypes.create_string_buffer(ERR_LEN)
    rc = lib.cudanet_k_gemm_f8(int(epi), int(bn), A.data_ptr(), W.data_ptr(), colscale.data_ptr(), bias.data_ptr(),
                               float(out_scale_inv), C.data_ptr(), M, N, K, C.stride(0), _stream(), err, ERR_LEN)
    if rc != 0:
        raise RuntimeError(f"cudanet_k_gemm_f8: {_msg(err)}")
    return C


def k_attention_f8(qkv, att, B, d, heads, mul, dll=None):
    """att (e4m3) = e4m3(attention(qkv) * mul), qkv bf16."""
    _e4m3(att, "att")
    lib = load(dll)
    err = ctypes.create_string_buffer(ERR_LEN)
    rc = lib.cudanet_k_attention_f8(qkv.data_ptr(), att.data_ptr(), B, d, heads, float(mul), _stream(), err, ERR_LEN)
    if rc != 0:
        raise RuntimeError(f"cudanet_k_attention_f8: {_msg(err)}")
    return att


def k_layernorm_f8(x, g, b, h, n, d, mul, row_stride=1, dll=None):
    """h (e4m3) = e4m3(LayerNorm(x) * mul), x float32 or bfloat16."""
    import torch
    _e4m3(h, "h")
    if x.dtype not in (torch.float32, torch.bfloat16):
        raise ValueError(f"x: float32 or bfloat16 only, got {x.dtype}")
    lib = load(dll)
    err = ctypes.create_string_buffer(ERR_LEN)
    rc = lib.cudanet_k_layernorm_f8(int(x.dtype == torch.bfloat16), x.data_ptr(), g.data_ptr(), b.data_ptr(),
                                    h.data_ptr(), n, d, row_stride, float(mul), _stream(), err, ERR_LEN)
    if rc != 0:
        raise RuntimeError(f"cudanet_k_layernorm_f8: {_msg(err)}")
    return h


# ------------------------------------------------------------------------------------------------ int8 operators
# These calls queue one kernel and return, so what a call costs on the host is most of what a small one costs (the
# library's part is about 3.5 us, the launch among it). Hence one straight condition in each that reads every attribute
# once; where it does not hold, _i8_matrix and _i8_vector find out why, or let the call through (a matrix of one column
# may have any step). The torch objects and the default library are looked up once a process, the reason buffer is kept
# by each thread.
class _I8Reason(threading.local):
    def __init__(self):
        self.buffer = ctypes.create_string_buffer(ERR_LEN)


_i8_reason = _I8Reason()
_i8_once = None


class _I8Once:
    """What the int8 calls need of torch: dtypes, their codes in the C ABI, the current device and stream."""

    def __init__(self):
        import torch
        self.int8, self.f32 = torch.int8, torch.float32
        self.types = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}
        self.on_device = torch.cuda.device
        # what torch's own generated code calls: a tenth of the cost of building a Stream object
        self.device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device
        self.stream = (getattr(torch._C, "_cuda_getCurrentRawStream", None)
                       or (lambda dev: torch.cuda.current_stream(dev).cuda_stream))
        self.lib = None

    def load(self, dll):
        """The library of `dll`; the default one (MAYFLY_CUDANET_DLL, else this package's) is looked up once."""
        if dll is not None:
            return load(dll)
        if self.lib is None:
            self.lib = load()
        return self.lib


def _i8_setup():
    global _i8_once
    if _i8_once is None:
        _i8_once = _I8Once()
    return _i8_once


def _i8_type(once, t, name):
    """The C ABI's code of a tensor's element type: 0 f16, 1 bf16, 2 f32."""
    code = once.types.get(t.dtype)
    if code is None:
        raise ValueError(f"{name}: float16, bfloat16 or float32 only, got {t.dtype}")
    return code


def _i8_matrix(t, name, shape, dev, dtype=None):
    """Raises unless t is a matrix of this shape and dtype (None: any) on device index dev with contiguous rows."""
    if dtype is not None and t.dtype is not dtype:
        raise ValueError(f"{name}: {dtype} only, got {t.dtype}")
    if len(t.shape) != 2 or t.shape != shape:
        raise ValueError(f"{name}: shape {tuple(t.shape)}, expected {tuple(shape) if len(shape) == 2 else 'a matrix'}")
    if dev < 0 or t.get_device() != dev:
        raise ValueError(f"{name}: on {t.device}, expected a tensor of one CUDA device with the others")
    if t.stride(1) != 1 and shape[1] > 1:
        raise ValueError(f"{name}: rows must be contiguous, got strides {t.stride()}")


def _i8_vector(once, t, name, n, dev):
    """Raises unless t is a contiguous float32 vector of n elements on device index dev."""
    if t.dtype is not once.f32:
        raise ValueError(f"{name}: float32 only, got {t.dtype}")
    if t.shape != (n,) or not t.is_contiguous():
        raise ValueError(f"{name}: shape {tuple(t.shape)} strides {t.stride()}, expected ({n},) contiguous")
    if t.get_device() != dev:
        raise ValueError(f"{name}: on {t.device}, expected a tensor of one CUDA device with the others")


def _i8_ints(**values):
    """Raises unless each fits the C ABI's 32-bit int: ctypes would pass its low 32 bits on."""
    for name, v in values.items():
        if not -2 ** 31 <= v < 2 ** 31:
            raise ValueError(f"{name}: {v} is over the 32 bits of the library's sizes")


def k_rmsnorm_i8(x, delta, g, out, q, scale, eps=1e-6, dll=None):
    """out = x + delta in x's type, and its RMS norm times g as int8 rows with a float32 scale each: q * scale stands
    for out / sqrt(mean(out^2) + eps) * g. x (M, D) float32, bfloat16 or float16; delta the same shape, of x's type or
    of any of the three where x is float32; out may be x (in place). delta and out None: the norm of x alone. q (M, D)
    int8, scale (M,) float32. Rows may have any pitch; asynchronous on the device's current stream. Returns (q,
    scale)."""
    once = _i8_once or _i8_setup()
    f32, shape, dev, xt = once.f32, x.shape, x.get_device(), _i8_type(once, x, "x")
    if len(shape) != 2:
        _i8_matrix(x, "x", shape, dev)
    (M, D), xs, qs = shape, x.stride(), q.stride()
    if (dev < 0 or M + D >= 2 ** 31 or xs[1] != 1 or q.dtype is not once.int8 or q.shape != shape or qs[1] != 1 or q.get_device() != dev
            or g.dtype is not f32 or g.shape != (D,) or g.get_device() != dev or not g.is_contiguous()
            or scale.dtype is not f32 or scale.shape != (M,) or scale.get_device() != dev
            or not scale.is_contiguous()):
        _i8_matrix(x, "x", shape, dev)
        _i8_matrix(q, "q", shape, dev, once.int8)
        _i8_vector(once, g, "g", D, dev)
        _i8_vector(once, scale, "scale", M, dev)
        _i8_ints(M=M, D=D)
    if delta is None:
        if out is not None:
            raise ValueError("out without delta: there is no sum to store")
        dt, ldd, ldo, dp, op = xt, 0, 0, None, None
    else:
        dt = _i8_type(once, delta, "delta")
        if out is None:
            raise ValueError("delta without out: out holds the sum (x itself: in place)")
        ds, os_ = delta.stride(), out.stride()
        if (delta.shape != shape or delta.get_device() != dev or ds[1] != 1 or out.dtype is not x.dtype
                or out.shape != shape or out.get_device() != dev or os_[1] != 1):
            _i8_matrix(delta, "delta", shape, dev)
            _i8_matrix(out, "out", shape, dev, x.dtype)
        ldd, ldo, dp, op = ds[0], os_[0], delta.data_ptr(), out.data_ptr()
    if once.device() != dev:
        with once.on_device(dev):
            return k_rmsnorm_i8(x, delta, g, out, q, scale, eps, dll)
    reason = _i8_reason.buffer
    if (once.lib if dll is None and once.lib else once.load(dll)).cudanet_k_rmsnorm_i8(
            xt, dt, x.data_ptr(), dp, g.data_ptr(), op, q.data_ptr(), scale.data_ptr(), M, D, xs[0], ldd, ldo,
            qs[0], eps, once.stream(dev), reason, ERR_LEN) != 0:
        raise RuntimeError(f"cudanet_k_rmsnorm_i8: {_msg(reason)}")
    return q, scale


def k_quant_i8(x, q, scale, dll=None):
    """x (M, D) float32, bfloat16 or float16 as int8 rows with a float32 scale each: scale = max |row| / 127, q * scale
    stands for x. A weight matrix (N, K) gets a scale for each output channel. Rows may have any pitch; asynchronous on
    the device's current stream. Returns (q, scale)."""
    once = _i8_once or _i8_setup()
    shape, dev, xt = x.shape, x.get_device(), _i8_type(once, x, "x")
    if len(shape) != 2:
        _i8_matrix(x, "x", shape, dev)
    (M, D), xs, qs = shape, x.stride(), q.stride()
    if (dev < 0 or M + D >= 2 ** 31 or xs[1] != 1 or q.dtype is not once.int8 or q.shape != shape or qs[1] != 1 or q.get_device() != dev
            or scale.dtype is not once.f32 or scale.shape != (M,) or scale.get_device() != dev
            or not scale.is_contiguous()):
        _i8_matrix(x, "x", shape, dev)
        _i8_matrix(q, "q", shape, dev, once.int8)
        _i8_vector(once, scale, "scale", M, dev)
        _i8_ints(M=M, D=D)
    if once.device() != dev:
        with once.on_device(dev):
            return k_quant_i8(x, q, scale, dll)
    reason = _i8_reason.buffer
    if (once.lib if dll is None and once.lib else once.load(dll)).cudanet_k_quant_i8(
            xt, x.data_ptr(), q.data_ptr(), scale.data_ptr(), M, D, xs[0], qs[0], once.stream(dev),
            reason, ERR_LEN) != 0:
        raise RuntimeError(f"cudanet_k_quant_i8: {_msg(reason)}")
    return q, scale


def k_gemm_i8(A, W, rowscale, colscale, bias, C, epi, kernel=-1, dll=None):
    """C = epilogue(A W^T * rowscale[m] * colscale[n] + bias[n]) with int8 A (M, K) and W (N, K), whose rows begin on
    16 bytes, the sum exact in int32, rowscale (M,), colscale (N,) and bias (N,) or None float32: epi 0 16-bit out, 1
    GELU and 16-bit out, 2 C += (float32), 3 float32 out. Asynchronous on the device's current stream. Returns C."""
    once = _i8_once or _i8_setup()
    i8, f32, sa, sw, dev, ct = once.int8, once.f32, A.shape, W.shape, A.get_device(), _i8_type(once, C, "C")
    if (ct == 2) != (epi >= 2):
        raise ValueError(f"C: epi {epi} writes {'float32' if epi >= 2 else 'float16 or bfloat16'}, got {C.dtype}")
    if len(sa) != 2 or len(sw) != 2 or sa[1] != sw[1]:
        raise ValueError(f"A and W: shapes {tuple(sa)} and {tuple(sw)}, expected (M, K) and (N, K)")
    M, K = sa
    N = sw[0]
    ta, tw, tc = A.stride(), W.stride(), C.stride()
    if (dev < 0 or M + N + K >= 2 ** 31 or (epi | kernel + 1) >> 7 or A.dtype is not i8 or ta[1] != 1 or W.dtype is not i8 or tw[1] != 1 or W.get_device() != dev
            or C.shape != (M, N) or tc[1] != 1 or C.get_device() != dev or rowscale.dtype is not f32
            or rowscale.shape != (M,) or rowscale.get_device() != dev or not rowscale.is_contiguous()
            or colscale.dtype is not f32 or colscale.shape != (N,) or colscale.get_device() != dev
            or not colscale.is_contiguous()):
        _i8_matrix(A, "A", sa, dev, i8)
        _i8_matrix(W, "W", sw, dev, i8)
        _i8_matrix(C, "C", (M, N), dev)
        _i8_vector(once, rowscale, "rowscale", M, dev)
        _i8_vector(once, colscale, "colscale", N, dev)
        _i8_ints(M=M, N=N, K=K, epi=epi, kernel=kernel)
    bp = None
    if bias is not None:
        if (bias.dtype is not f32 or bias.shape != (N,) or bias.get_device() != dev or not bias.is_contiguous()):
            _i8_vector(once, bias, "bias", N, dev)
        bp = bias.data_ptr()
    if once.device() != dev:
        with once.on_device(dev):
            return k_gemm_i8(A, W, rowscale, colscale, bias, C, epi, kernel, dll)
    reason = _i8_reason.buffer
    if (once.lib if dll is None and once.lib else once.load(dll)).cudanet_k_gemm_i8(
            ct & 1, epi, kernel, A.data_ptr(), W.data_ptr(), rowscale.data_ptr(), colscale.data_ptr(), bp,
            C.data_ptr(), M, N, K, ta[0], tw[0], tc[0], once.stream(dev), reason, ERR_LEN) != 0:
        raise RuntimeError(f"cudanet_k_gemm_i8: {_msg(reason)}")
    return C


def k_i8_check(stream=None, dll=None):
    """Wait for `stream` (a torch.cuda.Stream, default the current one) and raise if a bounded wait of a k_gemm_i8 call
    on its device has failed since the last check."""
    import torch
    s = stream if stream is not None else torch.cuda.current_stream()
    err = ctypes.create_string_buffer(ERR_LEN)
    with torch.cuda.device(s.device):
        rc = load(dll).cudanet_k_i8_check(ctypes.c_void_p(s.cuda_stream), err, ERR_LEN)
    if rc != 0:
        raise RuntimeError(f"cudanet_k_i8_check: {_msg(err)}")
