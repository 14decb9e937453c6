"""Safe wrappers over the C ABI of libcoli_b200.so — the role crates/colibri-backend/src/cuda.rs
plays for the reference (same call names, argument meaning and 1/0 return convention turned
into exceptions).  Host arrays are numpy, device arrays are torch CUDA tensors used purely as
memory (their ``data_ptr()`` is what crosses the ABI)."""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple

import numpy as np

from . import _lib
from .configs import FMT_E4M3_ROW, FMT_FP8_B128, FMT_MXFP4, FMT_NVFP4, SCORE_SOFTMAX, TYPE_BF16, TYPE_F16, TYPE_F32


class CudaError(RuntimeError):
    """A C-ABI call returned 0; the message is coli_cuda_last_error()."""


def _lib_():
    return _lib._lib or _lib.load()


def _check(ok: int, what: str) -> None:
    if not ok:
        msg = _lib_().coli_cuda_last_error().decode(errors="replace")
        raise CudaError(f"{what}: {msg}")


def _np_ptr(a: np.ndarray):
    assert a.flags["C_CONTIGUOUS"], "host arrays must be C-contiguous"
    return a.ctypes.data_as(C.c_void_p)


def init(devices=None) -> None:
    """coli_cuda_init (crates/colibri-backend/src/cuda.rs:400-430): idempotent per device set."""
    devices = [0] if devices is None else list(devices)
    arr = (C.c_int * len(devices))(*devices)
    _check(_lib_().coli_cuda_init(arr, len(devices)), "coli_cuda_init")


def shutdown() -> None:
    _lib_().coli_cuda_shutdown()


def device_count() -> int:
    return _lib_().coli_cuda_device_count()


def mem_info(device: int = 0):
    f, t = C.c_size_t(), C.c_size_t()
    _check(_lib_().coli_cuda_mem_info(device, C.byref(f), C.byref(t)), "coli_cuda_mem_info")
    return f.value, t.value


def stats(device: int = -1):
    n, b = C.c_size_t(), C.c_size_t()
    _lib_().coli_cuda_stats(device, C.byref(n), C.byref(b))
    return n.value, b.value


def device_sync(device: int = 0) -> None:
    _check(_lib_().coli_cuda_device_sync(device), "coli_cuda_device_sync")


def set_activation(oai: int = 0, alpha: float = 0.0, limit: float = 0.0) -> None:
    _lib_().coli_cuda_set_activation(oai, alpha, limit)


def sharding_fingerprint(num_nodes: int, n_experts: int, owner=None) -> int:
    if owner is None:
        return _lib_().coli_b200_sharding_fingerprint(num_nodes, n_experts, None)
    arr = np.ascontiguousarray(owner, dtype=np.uint32)
    return _lib_().coli_b200_sharding_fingerprint(num_nodes, n_experts, _np_ptr(arr))


class CudaTensor:
    """Persistent HBM copy of one quantised matrix W[O,I] (``ColiCudaTensor``)."""

    def __init__(self, handle: int, fmt: int, I: int, O: int, device: int):
        self.handle, self.fmt, self.I, self.O, self.device = handle, fmt, I, O, device

    # -- constructors ------------------------------------------------------------------
    @classmethod
    def wrap_nvfp4(cls, nibbles: np.ndarray, bscale: np.ndarray, gscale: float, I: int, O: int, device: int = 0):
        """coli_cuda_tensor_wrap_nvfp4: nibbles [O, ceil(I/2)] u8, bscale [O, ceil(I/16)] u8."""
        nibbles = np.ascontiguousarray(nibbles, dtype=np.uint8)
        bscale = np.ascontiguousarray(bscale, dtype=np.uint8)
        assert nibbles.size == O * ((I + 1) // 2) and bscale.size == O * ((I + 15) // 16)
        h = C.c_void_p()
        _check(_lib_().coli_cuda_tensor_wrap_nvfp4(C.byref(h), _np_ptr(nibbles), _np_ptr(bscale), float(gscale), I, O, device),
               "coli_cuda_tensor_wrap_nvfp4")
        return cls(h.value, FMT_NVFP4, I, O, device)

    @classmethod
    def wrap_mxfp4(cls, nibbles: np.ndarray, bscale: np.ndarray, gscale: float, I: int, O: int, device: int = 0):
        """coli_cuda_tensor_wrap_mxfp4: nibbles [O, ceil(I/2)] u8, bscale [O, ceil(I/32)] E8M0 bytes."""
        nibbles = np.ascontiguousarray(nibbles, dtype=np.uint8)
        bscale = np.ascontiguousarray(bscale, dtype=np.uint8)
        assert nibbles.size == O * ((I + 1) // 2) and bscale.size == O * ((I + 31) // 32)
        h = C.c_void_p()
        _check(_lib_().coli_cuda_tensor_wrap_mxfp4(C.byref(h), _np_ptr(nibbles), _np_ptr(bscale), float(gscale), I, O, device),
               "coli_cuda_tensor_wrap_mxfp4")
        return cls(h.value, FMT_MXFP4, I, O, device)

    @classmethod
    def upload(cls, codes: np.ndarray, scales: np.ndarray, fmt: int, I: int, O: int, device: int = 0):
        """coli_cuda_tensor_upload for the FP8 forms (fmt 4: row scales [O]; fmt 8: [ceil(O/128), ceil(I/128)])."""
        codes = np.ascontiguousarray(codes, dtype=np.uint8)
        scales = np.ascontiguousarray(scales, dtype=np.float32)
        assert codes.size == O * I
        want = O if fmt == FMT_E4M3_ROW else ((O + 127) // 128) * ((I + 127) // 128)
        assert scales.size == want
        h = C.c_void_p()
        _check(_lib_().coli_cuda_tensor_upload(C.byref(h), _np_ptr(codes), _np_ptr(scales), fmt, I, O, device),
               "coli_cuda_tensor_upload")
        return cls(h.value, fmt, I, O, device)

    @classmethod
    def from_device(cls, fmt: int, q, s, gscale: float, I: int, O: int, device: int = 0):
        """coli_b200_tensor_from_device: q, s are torch CUDA tensors in the reference layouts."""
        h = C.c_void_p()
        _check(_lib_().coli_b200_tensor_from_device(C.byref(h), fmt, q.data_ptr(), s.data_ptr(), float(gscale), I, O, device),
               "coli_b200_tensor_from_device")
        return cls(h.value, fmt, I, O, device)

    # -- accessors ---------------------------------------------------------------------
    def export(self):
        """Back to host in the reference layouts: (q u8, s u8|f32, gscale)."""
        I, O = self.I, self.O
        if self.fmt == FMT_NVFP4:
            q = np.empty((O, (I + 1) // 2), np.uint8)
            s = np.empty((O, (I + 15) // 16), np.uint8)
        elif self.fmt == FMT_MXFP4:
            q = np.empty((O, (I + 1) // 2), np.uint8)
            s = np.empty((O, (I + 31) // 32), np.uint8)
        elif self.fmt == FMT_FP8_B128:
            q = np.empty((O, I), np.uint8)
            s = np.empty(((O + 127) // 128, (I + 127) // 128), np.float32)
        else:
            q = np.empty((O, I), np.uint8)
            s = np.empty((O,), np.float32)
        g = C.c_float()
        _check(_lib_().coli_b200_tensor_export(self.handle, _np_ptr(q), _np_ptr(s), C.byref(g)), "coli_b200_tensor_export")
        return q, s, g.value

    def nbytes(self) -> int:
        return _lib_().coli_cuda_tensor_bytes(self.handle)

    def free(self) -> None:
        if self.handle:
            _lib_().coli_cuda_tensor_free(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass


# ---- device-side quantisers ------------------------------------------------------------------
def quantize_nvfp4_dev(w, device: int = 0):
    """f32 CUDA tensor [O,I] -> (nibbles u8 [O,ceil(I/2)], bscale u8 [O,ceil(I/16)], gscale)."""
    import torch

    O, I = w.shape
    assert w.dtype == torch.float32 and w.is_contiguous()
    nib = torch.empty((O, (I + 1) // 2), dtype=torch.uint8, device=w.device)
    bs = torch.empty((O, (I + 15) // 16), dtype=torch.uint8, device=w.device)
    g = C.c_float()
    _check(_lib_().coli_b200_quantize_nvfp4(device, w.data_ptr(), O, I, nib.data_ptr(), bs.data_ptr(), C.byref(g)),
           "coli_b200_quantize_nvfp4")
    return nib, bs, g.value


def quantize_fp8_b128_dev(w, device: int = 0):
    import torch

    O, I = w.shape
    assert w.dtype == torch.float32 and w.is_contiguous()
    codes = torch.empty((O, I), dtype=torch.uint8, device=w.device)
    sc = torch.empty(((O + 127) // 128, (I + 127) // 128), dtype=torch.float32, device=w.device)
    _check(_lib_().coli_b200_quantize_fp8_b128(device, w.data_ptr(), O, I, codes.data_ptr(), sc.data_ptr()),
           "coli_b200_quantize_fp8_b128")
    return codes, sc


# ---- 8-bit rows: e4m3 codes and an f32 scale per row and 128 columns ---------------------------------------
# A decode step makes these calls by the dozen and its kernels take a few microseconds each, so what stands around the C call
# reads every property of a tensor once (each costs 0.1 to 0.2 us).
class _Torch:
    """torch, looked up by the first device call: the host-array calls do without it."""

    def __init__(self):
        import torch

        self.types = {torch.float32: TYPE_F32, torch.float16: TYPE_F16, torch.bfloat16: TYPE_BF16}
        self.f32, self.i32, self.bf16, self.u8, self.empty = torch.float32, torch.int32, torch.bfloat16, torch.uint8, torch.empty
        # the handle of a device's current stream; the public way builds a Stream object for it (2.3 us against 0.1)
        self.stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda device: torch.cuda.current_stream(device).cuda_stream)


_torch = None


def _torch_() -> _Torch:
    global _torch
    if _torch is None:
        _torch = _Torch()
    return _torch


def _on(stream: int, device):
    """The current stream is `stream` (a raw handle) inside: what a call allocates there is handed out in that stream's order."""
    import torch

    return torch.cuda.stream(torch.cuda.ExternalStream(stream, device=device) if stream else torch.cuda.default_stream(device))


def _same_gpu(what: str, device: int, *tensors) -> None:
    """Raises unless every given tensor is on GPU `device` (-1: the host)."""
    for t in tensors:
        if t is not None and t.get_device() != device:
            raise ValueError(f"{what}: tensors on {t.device} and on {'cuda:%d' % device if device >= 0 else 'the host'}")
    if device < 0:
        raise ValueError(f"{what}: needs CUDA tensors")


def _rows_fp8(what: str, codes, scales, K: int):
    """(rows, bytes from row to row, strides of the scales) of a matrix in 8 bits, checked."""
    shape, stride = codes.shape, codes.stride()
    if len(shape) != 2 or shape[1] != K or codes.element_size() != 1 or (K > 1 and stride[1] != 1):
        raise ValueError(f"{what}: codes must be one byte each, [rows, {K}], columns next to each other")
    R = shape[0]
    if R > 1 << 30:  # (before ctypes cuts it to 32 bits)
        raise ValueError(f"{what}: {R} rows (at most 2^30)")
    if scales.shape != (R, (K + 127) // 128) or scales.dtype != _torch_().f32:
        raise ValueError(f"{what}: scales must be f32 [{R}, {(K + 127) // 128}], not {scales.dtype} {tuple(scales.shape)}")
    s_row, s_blk = scales.stride()
    ld = stride[0]
    if R < 2:  # (a single row may say anything)
        ld = (K + 15) // 16 * 16
    return R, ld, s_row, s_blk


def quantize_rows_fp8_dev(x, row_token=None, out=None, stream=None):
    """coli_b200_quantize_rows_fp8: rows of x (f32, f16 or bf16 [T,K] on the GPU, any row stride) -> (codes u8 [R,K],
    scales f32 [R, ceil(K/128)]), on the current torch stream or on `stream` (a raw handle); `init` need not come first.  With `row_token` (int32 [R]) row r is x[row_token[r]]; an entry
    outside [0,T) leaves the row as it was (uninitialised without `out`).  Fresh results have rows of codes that start on 16
    bytes and a block's scales next to each other; `out` = (codes, scales) are written in place whatever their strides, and
    the bytes behind a row's K codes become zero up to a multiple of 16, whatever they hold."""
    if stream is not None and x.is_cuda:
        with _on(stream, x.device):
            return quantize_rows_fp8_dev(x, row_token, out)
    th = _torch or _torch_()
    ty, shape, xs = th.types.get(x.dtype), x.shape, x.stride()
    if ty is None or len(shape) != 2 or shape[1] < 1 or (shape[1] > 1 and xs[1] != 1):
        raise ValueError("quantize_rows_fp8_dev: x must be f32, f16 or bf16 [T,K], columns next to each other")
    T, K = shape
    if T >= 1 << 31 or K >= 1 << 31:
        raise ValueError(f"quantize_rows_fp8_dev: x [{T}, {K}] is past 32 bits")
    if row_token is None:
        R, take = T, None
    elif row_token.dtype != th.i32 or row_token.dim() != 1 or not row_token.is_contiguous():
        raise ValueError("quantize_rows_fp8_dev: row_token must be contiguous int32 [rows]")
    else:
        R, take = row_token.shape[0], row_token.data_ptr()
    if out is None:
        codes = th.empty((R, (K + 15) // 16 * 16), dtype=th.u8, device=x.device)[:, :K]
        scales = th.empty(((K + 127) // 128, R), dtype=th.f32, device=x.device).t()
    else:
        codes, scales = out
    rows, ld, s_row, s_blk = _rows_fp8("quantize_rows_fp8_dev", codes, scales, K)
    if rows != R:
        raise ValueError(f"quantize_rows_fp8_dev: out has {rows} rows, not {R}")
    if out is not None and K % 16 and rows and codes.storage_offset() + (rows - 1) * ld + (K + 15) // 16 * 16 > codes.untyped_storage().nbytes():
        raise ValueError("quantize_rows_fp8_dev: out's codes need room up to a multiple of 16 bytes behind the last row")
    device = x.get_device()
    _same_gpu("quantize_rows_fp8_dev", device, codes, scales, row_token)
    if not _lib_().coli_b200_quantize_rows_fp8(device, x.data_ptr(), ty, xs[0], take, T, R, K, codes.data_ptr(), ld, scales.data_ptr(), s_row, s_blk,
                                               th.stream(device)):
        _check(0, "coli_b200_quantize_rows_fp8")
    return codes, scales


def matmul_fp8_dev(w: CudaTensor, codes, scales, out_dtype=None, out=None, stream=None):
    """coli_b200_matmul_fp8_dev: 8-bit rows [R, w.I] times a resident weight of format 8 -> [R, w.O] as `out_dtype` (bf16
    unless given) or into `out` (f32, f16 or bf16, any row stride), on the current torch stream or on `stream`."""
    if stream is not None and codes.is_cuda:
        with _on(stream, codes.device):
            return matmul_fp8_dev(w, codes, scales, out_dtype, out)
    th = _torch or _torch_()
    R, ld, s_row, s_blk = _rows_fp8("matmul_fp8_dev", codes, scales, w.I)
    O = w.O
    if out is None:
        out = th.empty((R, O), dtype=out_dtype or th.bf16, device=codes.device)
    ty, stride = th.types.get(out.dtype), out.stride()
    if out.shape != (R, O) or (O > 1 and stride[1] != 1) or ty is None or (out_dtype is not None and out_dtype != out.dtype):
        raise ValueError(f"matmul_fp8_dev: the result must be f32, f16 or bf16 [{R}, {O}], columns next to each other, of the type asked for")
    device = codes.get_device()
    _same_gpu("matmul_fp8_dev", device, scales, out)
    if device != w.device:
        raise ValueError(f"matmul_fp8_dev: the weight is on cuda:{w.device}, the rows on cuda:{device}")
    if not _lib_().coli_b200_matmul_fp8_dev(w.handle, codes.data_ptr(), ld, scales.data_ptr(), s_row, s_blk, R, out.data_ptr(), ty, stride[0],
                                            th.stream(device)):
        _check(0, "coli_b200_matmul_fp8_dev")
    return out


def fp8_check(device: int = 0) -> None:
    """Synchronise and raise if a matmul_fp8_dev on the device abandoned a bounded device-side wait."""
    _check(_lib_().coli_b200_fp8_check(device), "coli_b200_fp8_check")


# ---- routing from given logits -------------------------------------------------------------------------------
class Routing(NamedTuple):
    """What route_logits_dev answers: experts and weights of every token, and the rows its pairs take in expert order."""

    idx: object          # int32 [T,k], -1: none
    w: object            # f32 [T,k]
    expert_rows: object  # int32 [E]
    slot: object         # int32 [T,k], -1: none
    row_token: object    # int32 [T*k], -1 behind the last row


def route_logits_dev(logits, k: int, score: int = SCORE_SOFTMAX, select_bias=None, logit_bias=None, norm_topk: bool = False,
                     routed_scale: float = 1.0, n_group: int = 1, topk_group: int = 1, out=None, stream=None) -> Routing:
    """coli_b200_route_logits: router logits (f32, f16 or bf16 [T,E] on the GPU, rows E or more apart) -> Routing, on the current torch
    stream or on `stream`; `init` need not come first.  Biases are f32 [E]; -inf and NaN logits close an expert to a token; `out` is a Routing whose tensors are
    written in place."""
    if stream is not None and logits.is_cuda:
        with _on(stream, logits.device):
            return route_logits_dev(logits, k, score, select_bias, logit_bias, norm_topk, routed_scale, n_group, topk_group, out)
    th = _torch or _torch_()
    ty, shape, zs = th.types.get(logits.dtype), logits.shape, logits.stride()
    if ty is None or len(shape) != 2 or (shape[1] > 1 and zs[1] != 1):
        raise ValueError("route_logits_dev: logits must be f32, f16 or bf16 [T,E], experts next to each other")
    T, E = shape
    if T > 1 << 20 or E > 512:
        raise ValueError(f"route_logits_dev: logits [{T}, {E}] (T <= 2^20, E <= 512)")
    if not -(1 << 31) < min(k, score, n_group, topk_group) <= max(k, score, n_group, topk_group) < 1 << 31:  # (before ctypes cuts them)
        raise ValueError(f"route_logits_dev: k={k}, score={score}, n_group={n_group} or topk_group={topk_group} is past 32 bits")
    for name, b in (("select_bias", select_bias), ("logit_bias", logit_bias)):
        if b is not None and (b.dtype != th.f32 or b.numel() != E or not b.is_contiguous()):
            raise ValueError(f"route_logits_dev: {name} must be contiguous f32 [{E}]")
    if out is None:
        new = lambda dtype, *n: th.empty(n, dtype=dtype, device=logits.device)  # noqa: E731
        out = Routing(new(th.i32, T, k), new(th.f32, T, k), new(th.i32, E), new(th.i32, T, k), new(th.i32, T * k))
    else:
        if type(out) is not Routing:
            out = Routing(*out)
        pairs = (T, k)
        for name, t, want in zip(Routing._fields, out, (pairs, pairs, (E,), pairs, (T * k,))):
            if t.shape != want or t.dtype != (th.f32 if name == "w" else th.i32) or not t.is_contiguous():
                raise ValueError(f"route_logits_dev: out.{name} must be contiguous {'f32' if name == 'w' else 'int32'} {list(want)}")
    device = logits.get_device()
    _same_gpu("route_logits_dev", device, select_bias, logit_bias, *out)
    lib = _lib_()
    n = lib.coli_b200_route_logits_workspace(T, E)
    work = th.empty(n, dtype=th.u8, device=logits.device) if n else None
    if not lib.coli_b200_route_logits(device, logits.data_ptr(), ty, zs[0] if T > 1 else E, None if select_bias is None else select_bias.data_ptr(),
                                      None if logit_bias is None else logit_bias.data_ptr(), T, E, k, score, norm_topk, routed_scale, n_group,
                                      topk_group, out.idx.data_ptr(), out.w.data_ptr(), out.expert_rows.data_ptr(), out.slot.data_ptr(),
                                      out.row_token.data_ptr(), None if work is None else work.data_ptr(), th.stream(device)):
        _check(0, "coli_b200_route_logits")
    return out


# ---- the reference's host-pointer expert calls ---------------------------------------------------
def expert_mlp_nvfp4(gate: CudaTensor, up: CudaTensor, down: CudaTensor, x: np.ndarray) -> np.ndarray:
    """coli_cuda_expert_mlp_nvfp4 (cuda.rs:833-880): x, y host f32 [S, D]."""
    x = np.ascontiguousarray(x, dtype=np.float32)
    y = np.empty_like(x)
    _check(_lib_().coli_cuda_expert_mlp_nvfp4(gate.handle, up.handle, down.handle, _np_ptr(y), _np_ptr(x), x.shape[0]),
           "coli_cuda_expert_mlp_nvfp4")
    return y


def expert_mlp_fp8(gate: CudaTensor, up: CudaTensor, down: CudaTensor, x: np.ndarray) -> np.ndarray:
    x = np.ascontiguousarray(x, dtype=np.float32)
    y = np.empty_like(x)
    _check(_lib_().coli_cuda_expert_mlp_fp8(gate.handle, up.handle, down.handle, _np_ptr(y), _np_ptr(x), x.shape[0]),
           "coli_cuda_expert_mlp_fp8")
    return y


def expert_group_nvfp4(gates, ups, downs, rows, x: np.ndarray) -> np.ndarray:
    """coli_cuda_expert_group_nvfp4 (cuda.rs:1020-1067): x holds sum(rows) rows in expert order."""
    n = len(rows)
    x = np.ascontiguousarray(x, dtype=np.float32)
    y = np.empty_like(x)
    mk = lambda ts: (C.c_void_p * n)(*[t.handle for t in ts])
    r = (C.c_int * n)(*[int(v) for v in rows])
    _check(_lib_().coli_cuda_expert_group_nvfp4(mk(gates), mk(ups), mk(downs), r, n, _np_ptr(y), _np_ptr(x)),
           "coli_cuda_expert_group_nvfp4")
    return y


def expert_mlp_mxfp4(gate: CudaTensor, up: CudaTensor, down: CudaTensor, x: np.ndarray) -> np.ndarray:
    """coli_cuda_expert_mlp_mxfp4 (cuda.rs:92-99): fmt 6 on all three; x, y host f32 [S, D]."""
    x = np.ascontiguousarray(x, dtype=np.float32)
    y = np.empty_like(x)
    _check(_lib_().coli_cuda_expert_mlp_mxfp4(gate.handle, up.handle, down.handle, _np_ptr(y), _np_ptr(x), x.shape[0]),
           "coli_cuda_expert_mlp_mxfp4")
    return y


def expert_group_mxfp4(gates, ups, downs, rows, x: np.ndarray) -> np.ndarray:
    """coli_cuda_expert_group_mxfp4 (cuda.rs:212-220): x holds sum(rows) rows in expert order."""
    n = len(rows)
    x = np.ascontiguousarray(x, dtype=np.float32)
    y = np.empty_like(x)
    mk = lambda ts: (C.c_void_p * n)(*[t.handle for t in ts])
    r = (C.c_int * n)(*[int(v) for v in rows])
    _check(_lib_().coli_cuda_expert_group_mxfp4(mk(gates), mk(ups), mk(downs), r, n, _np_ptr(y), _np_ptr(x)),
           "coli_cuda_expert_group_mxfp4")
    return y


def scratch_bytes(device: int = -1) -> int:
    """coli_cuda_scratch_bytes (backend_cuda.h:48-51)."""
    return int(_lib_().coli_cuda_scratch_bytes(device))


def group_stats() -> dict:
    """coli_cuda_group_stats (backend_cuda.h:52-53): totals over the grouped expert calls since load."""
    c, e, r = C.c_uint64(), C.c_uint64(), C.c_uint64()
    a, b, d = C.c_double(), C.c_double(), C.c_double()
    _lib_().coli_cuda_group_stats(C.byref(c), C.byref(e), C.byref(r), C.byref(a), C.byref(b), C.byref(d))
    return dict(calls=c.value, experts=e.value, rows=r.value, h2d_ms=a.value, kernel_ms=b.value, d2h_ms=d.value)


class F32Matmul:
    """coli_cuda_matmul with fmt 0 — the router GEMM of crates/colibri-engine/src/gpu.rs:2219-2249.
    Keeps the ``slot`` the reference threads through the call so W is uploaded once."""

    def __init__(self, w: np.ndarray, device: int = 0):
        self.w = np.ascontiguousarray(w, dtype=np.float32)
        self.O, self.I = self.w.shape
        self.device = device
        self.slot = C.c_void_p()

    def __call__(self, x: np.ndarray) -> np.ndarray:
        x = np.ascontiguousarray(x, dtype=np.float32)
        y = np.empty((x.shape[0], self.O), np.float32)
        _check(_lib_().coli_cuda_matmul(C.byref(self.slot), _np_ptr(y), _np_ptr(x), _np_ptr(self.w), None, 0,
                                        x.shape[0], self.I, self.O, self.device), "coli_cuda_matmul")
        return y

    def free(self):
        if self.slot.value:
            _lib_().coli_cuda_tensor_free(self.slot)
            self.slot = C.c_void_p()


def expert_mlp(gate: CudaTensor, up: CudaTensor, down: CudaTensor, x: np.ndarray) -> np.ndarray:
    """coli_cuda_expert_mlp (backend_cuda.h:107-109): any resident expert format."""
    x = np.ascontiguousarray(x, dtype=np.float32)
    y = np.empty_like(x)
    _check(_lib_().coli_cuda_expert_mlp(gate.handle, up.handle, down.handle, _np_ptr(y), _np_ptr(x), x.shape[0]),
           "coli_cuda_expert_mlp")
    return y


def expert_group(gates, ups, downs, rows, x: np.ndarray) -> np.ndarray:
    """coli_cuda_expert_group (backend_cuda.h:136-140): x holds sum(rows) rows in expert order."""
    n = len(rows)
    x = np.ascontiguousarray(x, dtype=np.float32)
    y = np.empty_like(x)
    mk = lambda ts: (C.c_void_p * n)(*[t.handle for t in ts])
    r = (C.c_int * n)(*[int(v) for v in rows])
    _check(_lib_().coli_cuda_expert_group(mk(gates), mk(ups), mk(downs), r, n, _np_ptr(y), _np_ptr(x)), "coli_cuda_expert_group")
    return y


class Nvfp4Matmul:
    """coli_cuda_matmul_nvfp4 (backend_cuda.h:127-129): y = x @ W^T for one NVFP4 matrix given as the
    container's host arrays; the slot keeps the HBM copy between calls."""

    def __init__(self, nibbles: np.ndarray, bscale: np.ndarray, gscale: float, O: int, I: int, device: int = 0):
        self.nib = np.ascontiguousarray(nibbles, dtype=np.uint8)
        self.bs = np.ascontiguousarray(bscale, dtype=np.uint8)
        self.g, self.O, self.I, self.device = float(gscale), O, I, device
        self.slot = C.c_void_p()

    def __call__(self, x: np.ndarray) -> np.ndarray:
        x = np.ascontiguousarray(x, dtype=np.float32)
        y = np.empty((x.shape[0], self.O), np.float32)
        _check(_lib_().coli_cuda_matmul_nvfp4(C.byref(self.slot), _np_ptr(y), _np_ptr(x), _np_ptr(self.nib), _np_ptr(self.bs),
                                              self.g, x.shape[0], self.I, self.O, self.device), "coli_cuda_matmul_nvfp4")
        return y

    def free(self):
        if self.slot.value:
            _lib_().coli_cuda_tensor_free(self.slot)
            self.slot = C.c_void_p()


def expert_group_relu2(ups, downs, rows, x: np.ndarray, seg: bool = False) -> np.ndarray:
    """coli_cuda_expert_group_nvfp4_relu2 / coli_cuda_expert_seg_nvfp4_relu2 (backend_cuda.h:152-160):
    gateless experts, y = down(relu(up x)^2); x holds sum(rows) rows in expert order."""
    n = len(rows)
    x = np.ascontiguousarray(x, dtype=np.float32)
    y = np.empty_like(x)
    mk = lambda ts: (C.c_void_p * n)(*[t.handle for t in ts])
    r = (C.c_int * n)(*[int(v) for v in rows])
    fn = _lib_().coli_cuda_expert_seg_nvfp4_relu2 if seg else _lib_().coli_cuda_expert_group_nvfp4_relu2
    _check(fn(mk(ups), mk(downs), r, n, _np_ptr(y), _np_ptr(x)), "coli_cuda_expert_group_nvfp4_relu2")
    return y


def expert_mlp_relu2(up: CudaTensor, down: CudaTensor, x: np.ndarray, exact: bool = False) -> np.ndarray:
    """coli_cuda_expert_mlp_nvfp4_relu2 (backend_cuda.h:131-132)."""
    x = np.ascontiguousarray(x, dtype=np.float32)
    y = np.empty_like(x)
    _check(_lib_().coli_cuda_expert_mlp_nvfp4_relu2(up.handle, down.handle, _np_ptr(y), _np_ptr(x), x.shape[0], int(exact)),
           "coli_cuda_expert_mlp_nvfp4_relu2")
    return y
