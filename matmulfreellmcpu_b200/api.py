"""Python front of the C ABI, mirroring the reference engine's C++ API.

``Model`` mirrors ``mmfree::Model`` (matmulfreellmCPU cpp/include/mmfree/model.hpp:33-80)
plus the step-wise serving session; the kernel functions mirror ``mmfree::bitlinear``,
``bitlinear_cluster``, ``rmsnorm``, ``swiglu``, ``hgrn_scan`` and ``rmsnorm_swishgate``
(kernels.hpp:29-68) on CUDA tensors (torch is used only to hold device memory and streams).
Beside them stand the operators of a block with a selective scan as its token mixer
(``add_rmsnorm_quant``, ``int4_matvec``, ``causal_conv``, ``selective_scan`` and the
single-token forms), which the reference lacks.
Errors raise :class:`MmfreeError`, the counterpart of the reference's std::runtime_error.
"""
from __future__ import annotations

import ctypes as C
from dataclasses import dataclass

import numpy as np

from ._lib import (ACT_FIXED_Q510, ACT_FLOAT, E_INVALID, T_BF16, T_E4M3, T_F16, T_F32,  # noqa: F401
                   T_S8, ConvArgs, MmfreeError, SsmArgs, check, lib)

ActQuant = {"float": ACT_FLOAT, "fixed": ACT_FIXED_Q510}


def _aq(mode) -> int:
    if isinstance(mode, str):
        return ActQuant[mode]
    return int(mode)


def _ptr(t) -> int | None:
    return None if t is None else t.data_ptr()


def _stream(stream=None) -> int | None:
    if stream is not None:
        return stream.cuda_stream
    import torch
    return torch.cuda.current_stream().cuda_stream


def _i64(a) -> np.ndarray:
    return np.ascontiguousarray(np.asarray(a, dtype=np.int64))


@dataclass
class Config:  # mmfree::Config (config.hpp:8-21)
    vocab_size: int
    hidden_size: int
    num_hidden_layers: int
    num_heads: int
    expand_ratio: int
    intermediate_size: int
    use_lower_bound: bool
    use_short_conv: bool
    rms_norm_eps: float


class _CConfig(C.Structure):
    _fields_ = [(n, C.c_size_t) for n in ("vocab_size", "hidden_size", "num_hidden_layers",
                                           "num_heads", "expand_ratio", "intermediate_size")] + \
               [("use_lower_bound", C.c_int), ("use_short_conv", C.c_int),
                ("rms_norm_eps", C.c_float)]


def _config(c: "_CConfig") -> Config:
    return Config(c.vocab_size, c.hidden_size, c.num_hidden_layers, c.num_heads, c.expand_ratio,
                  c.intermediate_size, bool(c.use_lower_bound), bool(c.use_short_conv),
                  float(c.rms_norm_eps))


def blob_config(path: str) -> Config:
    """Header of a model.mmfree blob (host only, no GPU needed)."""
    c = _CConfig()
    check(lib().mmfree_cuda_blob_config(path.encode(), C.byref(c)))
    return _config(c)


class Model:
    """Device-resident HGRN-Bit model opened from a ``model.mmfree`` blob."""

    def __init__(self, blob_path: str, act_quant="fixed", frac_bits: int = 10, device: int = 0):
        h = C.c_void_p()
        check(lib().mmfree_cuda_model_open(blob_path.encode(), device, _aq(act_quant), frac_bits,
                                           C.byref(h)))
        self._h = h
        c = _CConfig()
        check(lib().mmfree_cuda_model_config(self._h, C.byref(c)))
        self.config = _config(c)
        self.device = device

    @classmethod
    def open_tp(cls, blob_path: str, act_quant, rank: int, world: int, nccl_id: bytes,
                frac_bits: int = 10, device: int = 0) -> "Model":
        """Rank ``rank`` of a ``world``-way tensor-parallel prefill handle (collective: every
        rank opens its handle with the same NCCL id; see ``matmulfreellmcpu_b200.tp``)."""
        if len(nccl_id) != 128:
            raise ValueError("an NCCL unique id has 128 bytes")
        self = cls.__new__(cls)
        h = C.c_void_p()
        buf = (C.c_ubyte * 128).from_buffer_copy(nccl_id)
        check(lib().mmfree_cuda_model_open_tp(blob_path.encode(), device, _aq(act_quant), frac_bits,
                                              rank, world, buf, C.byref(h)))
        self._h = h
        c = _CConfig()
        check(lib().mmfree_cuda_model_config(self._h, C.byref(c)))
        self.config = _config(c)
        self.device = device
        return self

    def close(self) -> None:
        if getattr(self, "_h", None):
            lib().mmfree_cuda_model_close(self._h)
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

    @property
    def weight_bytes(self) -> int:
        return lib().mmfree_cuda_model_weight_bytes(self._h)

    def generate(self, ids, new_tokens: int, eos_id: int = -1, temperature: float = 0.0,
                 top_k: int = 0, seed: int = 0) -> np.ndarray:
        """Model::generate: prompt + generated ids."""
        ids = _i64(ids)
        out = np.empty(ids.size + new_tokens, np.int64)
        n = C.c_size_t()
        check(lib().mmfree_cuda_generate(self._h, ids.ctypes.data, ids.size, new_tokens, eos_id,
                                         temperature, top_k, seed, out.ctypes.data, out.size,
                                         C.byref(n)))
        return out[:n.value]

    def forward(self, ids) -> np.ndarray:
        """Model::forward: logits [T, vocab] from a zero state."""
        ids = _i64(ids)
        lg = np.empty((ids.size, self.config.vocab_size), np.float32)
        check(lib().mmfree_cuda_forward(self._h, ids.ctypes.data, ids.size, lg.ctypes.data))
        return lg

    def forward_trace(self, ids):
        """(logits [T, V], trace [1 + 3L, T, H]): embeddings, then per layer the recurrence
        output, the residual after o_proj and the layer output."""
        ids = _i64(ids)
        c = self.config
        lg = np.empty((ids.size, c.vocab_size), np.float32)
        tr = np.empty((1 + 3 * c.num_hidden_layers, ids.size, c.hidden_size), np.float32)
        check(lib().mmfree_cuda_forward_trace(self._h, ids.ctypes.data, ids.size, lg.ctypes.data,
                                              tr.ctypes.data))
        return lg, tr

    def forward_last(self, ids) -> np.ndarray:
        ids = _i64(ids)
        lg = np.empty(self.config.vocab_size, np.float32)
        check(lib().mmfree_cuda_forward_last(self._h, ids.ctypes.data, ids.size, lg.ctypes.data))
        return lg

    @staticmethod
    def _prompts(prompts):
        ps = [_i64(p) for p in prompts]
        arr = (C.c_void_p * len(ps))(*[p.ctypes.data for p in ps])
        lens = (C.c_size_t * len(ps))(*[p.size for p in ps])
        return ps, arr, lens

    def generate_serve(self, prompts, new_tokens: int, eos_id: int = -1,
                       temperature: float = 0.0, top_k: int = 0, seed: int = 0):
        """Model::generate_serve: list of B full id streams."""
        ps, arr, lens = self._prompts(prompts)
        B = len(ps)
        stride = max(p.size for p in ps) + max(new_tokens, 1)
        out = np.zeros((B, stride), np.int64)
        out_lens = np.zeros(B, np.uint64)
        check(lib().mmfree_cuda_generate_serve(self._h, B, arr, lens, new_tokens, eos_id,
                                               temperature, top_k, seed, out.ctypes.data, stride,
                                               out_lens.ctypes.data))
        return [out[b, :int(out_lens[b])] for b in range(B)]

    def serve_begin(self, prompts) -> np.ndarray:
        ps, arr, lens = self._prompts(prompts)
        first = np.empty(len(ps), np.int64)
        check(lib().mmfree_cuda_serve_begin(self._h, len(ps), arr, lens, first.ctypes.data))
        self._serve_b = len(ps)
        return first

    def serve_step(self, in_ids, out=None) -> np.ndarray:
        in_ids = _i64(in_ids)
        out = np.empty(in_ids.size, np.int64) if out is None else out
        check(lib().mmfree_cuda_serve_step(self._h, in_ids.ctypes.data, out.ctypes.data))
        return out

    def serve_step_ptr(self, in_ptr: int, out_ptr: int) -> None:
        """serve_step on raw host pointers (pinned buffers)."""
        check(lib().mmfree_cuda_serve_step(self._h, in_ptr, out_ptr))

    def serve_run(self, steps: int) -> np.ndarray:
        out = np.empty((self._serve_b, steps), np.int64)
        check(lib().mmfree_cuda_serve_run(self._h, steps, out.ctypes.data))
        return out

    def serve_end(self) -> None:
        check(lib().mmfree_cuda_serve_end(self._h))

    @property
    def stream_ptr(self) -> int:
        """cudaStream_t of every kernel this model launches (for CUDA-event timing)."""
        return lib().mmfree_cuda_model_stream(self._h)

    def serve_profile(self, steps: int) -> dict:
        """Per kernel class: {name: dict(ms, launches, bytes, ops)} over ``steps`` steps."""
        from ._lib import KernelStats
        buf = (KernelStats * 16)()
        n = C.c_int()
        check(lib().mmfree_cuda_serve_profile(self._h, steps, buf, 16, C.byref(n)))
        return {buf[i].name.decode(): dict(ms=buf[i].ms, launches=buf[i].launches,
                                           bytes=buf[i].bytes, ops=buf[i].ops)
                for i in range(n.value)}


# ---- kernels on CUDA tensors -----------------------------------------------------------------

def packed_bytes(out_dim: int, in_dim: int) -> int:
    return lib().mmfree_cuda_packed_bytes(out_dim, in_dim)


def pack_ternary_host(wq: np.ndarray) -> np.ndarray:
    """int8 [out, in] -> packed uint8 bytes (host)."""
    wq = np.ascontiguousarray(wq, np.int8)
    out = np.empty(packed_bytes(*wq.shape), np.uint8)
    check(lib().mmfree_cuda_pack_ternary_host(out.ctypes.data, wq.ctypes.data, *wq.shape))
    return out


def repack_ternary(wq, stream=None):
    """int8 CUDA tensor [out, in] -> packed uint8 CUDA tensor."""
    import torch
    out = torch.empty(packed_bytes(*wq.shape), dtype=torch.uint8, device=wq.device)
    check(lib().mmfree_cuda_repack_ternary(out.data_ptr(), wq.contiguous().data_ptr(),
                                           wq.shape[0], wq.shape[1], _stream(stream)))
    return out


def bitlinear(x, norm_weight, wpacked, scale_w: float, out_dim: int, eps: float = 1e-6,
              act_quant="fixed", frac_bits: int = 10, want_norm: bool = False,
              want_acc: bool = False, stream=None):
    """mmfree::bitlinear on CUDA tensors; returns (out, acc or None, norm or None)."""
    import torch
    rows, in_dim = x.shape
    out = torch.empty(rows, out_dim, dtype=torch.float32, device=x.device)
    norm = torch.empty_like(x) if want_norm else None
    acc = torch.empty(rows, out_dim, dtype=torch.int32, device=x.device) if want_acc else None
    check(lib().mmfree_cuda_bitlinear(out.data_ptr(), x.data_ptr(), norm_weight.data_ptr(),
                                      wpacked.data_ptr(), scale_w, rows, in_dim, out_dim, eps,
                                      _ptr(norm), _aq(act_quant), frac_bits, _ptr(acc),
                                      _stream(stream)))
    return out, acc, norm


def nccl_unique_id() -> bytes:
    """128 bytes that identify a new NCCL communicator (rank 0 makes it, every rank uses it)."""
    buf = (C.c_ubyte * 128)()
    check(lib().mmfree_cuda_nccl_unique_id(buf))
    return bytes(buf)


def kernel_status(stream=None) -> None:
    """Synchronizes ``stream`` and raises MmfreeError (code E_TIMEOUT) when a kernel of an
    asynchronous entry point (bitlinear, bitlinear_cluster, bitlinear_noalloc) gave up a
    bounded wait since the last check; the recorded error is cleared."""
    check(lib().mmfree_cuda_kernel_status(_stream(stream)))


def set_wait_limit(polls: int) -> None:
    """Diagnostic: polls of the BitLinear prologue's row wait before it gives up (negative =
    default); 0 makes the staged waits give up at once."""
    lib().mmfree_cuda_set_wait_limit(int(polls))


def bitlinear_cluster(x, norm_weights, wpacked, scale_w, out_dim: int, eps: float = 1e-6,
                      frac_bits: int = 10, want_acc: bool = False, stream=None):
    import torch
    rows, in_dim = x.shape
    k = len(norm_weights)
    outs = [torch.empty(rows, out_dim, dtype=torch.float32, device=x.device) for _ in range(k)]
    acc = torch.empty(k, rows, out_dim, dtype=torch.int32, device=x.device) if want_acc else None
    o = (C.c_void_p * k)(*[t.data_ptr() for t in outs])
    n = (C.c_void_p * k)(*[t.data_ptr() for t in norm_weights])
    w = (C.c_void_p * k)(*[t.data_ptr() for t in wpacked])
    s = (C.c_float * k)(*[float(v) for v in scale_w])
    check(lib().mmfree_cuda_bitlinear_cluster(o, x.data_ptr(), n, w, s, k, rows, in_dim, out_dim,
                                              eps, frac_bits, _ptr(acc), _stream(stream)))
    return outs, acc


def ternary_matmul(x_codes, wpacked, out_dim: int, stream=None):
    """TernaryBackend::matmul_batch: int32 codes [b, N] -> int32 acc [b, M]."""
    import torch
    b, n = x_codes.shape
    acc = torch.empty(b, out_dim, dtype=torch.int32, device=x_codes.device)
    check(lib().mmfree_cuda_ternary_matmul(acc.data_ptr(), x_codes.data_ptr(), wpacked.data_ptr(),
                                           n, out_dim, b, _stream(stream)))
    return acc


def rmsnorm(x, weight, eps: float = 1e-6, stream=None):
    import torch
    y = torch.empty_like(x)
    check(lib().mmfree_cuda_rmsnorm(y.data_ptr(), x.data_ptr(), weight.data_ptr(), x.shape[0],
                                    x.shape[1], eps, _stream(stream)))
    return y


def swiglu(a, b, stream=None):
    import torch
    out = torch.empty_like(a)
    check(lib().mmfree_cuda_swiglu(out.data_ptr(), a.data_ptr(), b.data_ptr(), a.numel(),
                                   _stream(stream)))
    return out


def hgrn_scan(i, f, state=None, stream=None):
    """mmfree::hgrn_scan; ``state`` (CUDA tensor [D]) is updated in place when given."""
    import torch
    out = torch.empty_like(i)
    T, D = i.shape
    check(lib().mmfree_cuda_hgrn_scan(out.data_ptr(), i.data_ptr(), f.data_ptr(), T, D,
                                      _ptr(state), _stream(stream)))
    return out


def rmsnorm_swishgate(g, o, weight, eps: float = 1e-6, stream=None):
    import torch
    out = torch.empty_like(g)
    check(lib().mmfree_cuda_rmsnorm_swishgate(out.data_ptr(), g.data_ptr(), o.data_ptr(),
                                              weight.data_ptr(), g.shape[0], g.shape[1], eps,
                                              _stream(stream)))
    return out


# ---- operators of a recurrent block ------------------------------------------------------------
# Rows may be slices of wider rows (any row pitch, contiguous elements). With ``stream`` the
# call runs on that stream and its outputs belong to it, as torch tensors made under
# ``torch.cuda.stream(stream)`` do; without, on the tensors' device's current stream.

_TYPES: dict = {}


def _type_of(dtype) -> int | None:
    if not _TYPES:
        import torch
        _TYPES.update({torch.float32: T_F32, torch.bfloat16: T_BF16, torch.float16: T_F16,
                       torch.int8: T_S8, torch.float8_e4m3fn: T_E4M3})
    return _TYPES.get(dtype)


def _need(ok, what: str) -> None:
    if not ok:
        raise MmfreeError(E_INVALID, what)


def _row_type(t, name: str) -> int:
    code = _type_of(t.dtype)
    _need(code is not None and code <= T_F16, f"{name} must be float32, bfloat16 or float16")
    return code


def _pitch(t, name: str, rows: int, cols: int, dtype, device) -> int:
    """Row pitch of a [rows, cols] operand, checked."""
    _need(t.device == device, f"{name} is on {t.device}, not on {device}")
    _need(t.dtype == dtype, f"{name} must be {dtype}, not {t.dtype}")
    _need(t.dim() == 2 and t.shape[0] == rows and t.shape[1] == cols,
          f"{name} must be [{rows}, {cols}], not {list(t.shape)}")
    s = t.stride()
    _need(s[1] == 1 or cols <= 1, f"{name}'s rows must be contiguous")
    return s[0]


def _dense(t, name: str, shape: tuple, dtype, device) -> None:
    _need(t.device == device, f"{name} is on {t.device}, not on {device}")
    _need(t.dtype == dtype, f"{name} must be {dtype}, not {t.dtype}")
    _need(tuple(t.shape) == shape and t.is_contiguous(),
          f"{name} must be a contiguous {list(shape)}, not {list(t.shape)}")


def _span(t) -> tuple[int, int]:
    """The bytes from a tensor's first to behind its last element."""
    last = sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
    return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size() if t.numel() else t.data_ptr()


def _apart(a, a_name: str, b, b_name: str) -> None:
    if b is not None:
        (a0, a1), (b0, b1) = _span(a), _span(b)
        _need(a1 <= b0 or b1 <= a0, f"{a_name} overlaps {b_name}")


class _On:
    """The device and stream of one call: makes its outputs there and runs the entry point."""

    __slots__ = ("device", "stream", "other")

    def __init__(self, x, stream):
        import torch
        _need(x.is_cuda, "the tensors must be on a CUDA device")
        self.device = x.device
        self.other = stream
        if stream is None:
            self.stream = torch.cuda.current_stream(self.device).cuda_stream
        else:
            _need(stream.device == self.device, f"the stream is on {stream.device}, not on {self.device}")
            self.stream = stream.cuda_stream

    def empty(self, *shape, dtype):
        import torch
        if self.other is None:
            return torch.empty(shape, dtype=dtype, device=self.device)
        with torch.cuda.stream(self.other):
            return torch.empty(shape, dtype=dtype, device=self.device)

    def run(self, entry, *args, held=()) -> None:
        import torch
        if self.other is not None:  # the caller's allocator streams may differ from this one
            for t in held:
                if t is not None:
                    t.record_stream(self.other)
        if torch.cuda.current_device() == self.device.index:
            check(entry(*args, self.stream))
        else:
            with torch.cuda.device(self.device):
                check(entry(*args, self.stream))


def add_rmsnorm_quant(x, weight, residual=None, eps: float = 1e-6, code: str = "int8", group: int = 0,
                      stream=None):
    """``residual += x`` (in place, when given), then the RMS norm of it (of ``x`` without) times
    ``weight`` as 8-bit codes: returns ``(codes, scales)`` with norm ~ codes * scales.

    ``x`` and ``residual`` [rows, cols] float32, bfloat16 or float16, ``weight`` [cols] float32.
    ``code``: "int8" (the exact quotient by the scale, half to even) or "e4m3"
    (torch.float8_e4m3fn). ``group``: columns of a scale, 32, 64 or 128, or 0 for one scale a
    row; ``scales`` is float32 [rows, ceil(cols / group)], a row's [rows, 1]."""
    import torch
    kind = _row_type(x, "x")
    _need(x.dim() == 2, "x must be [rows, cols]")
    rows, cols = x.shape
    on = _On(x, stream)
    ldx = _pitch(x, "x", rows, cols, x.dtype, on.device)
    _dense(weight, "weight", (cols,), torch.float32, on.device)
    _need(code in ("int8", "e4m3"), "code must be 'int8' or 'e4m3'")
    _need(group in (0, 32, 64, 128), "group must be 0, 32, 64 or 128")
    ldr = 0
    if residual is not None:
        ldr = _pitch(residual, "residual", rows, cols, x.dtype, on.device)
        _apart(residual, "residual", x, "x")
        _apart(residual, "residual", weight, "weight")
    codes = on.empty(rows, cols, dtype=torch.int8 if code == "int8" else torch.float8_e4m3fn)
    scales = on.empty(rows, -(-cols // group) if group else 1, dtype=torch.float32)
    on.run(lib().mmfree_cuda_add_rmsnorm_quant, codes.data_ptr(), scales.data_ptr(), x.data_ptr(), ldx,
           _ptr(residual), ldr, weight.data_ptr(), rows, cols, eps, kind,
           T_S8 if code == "int8" else T_E4M3, group, held=(x, residual, weight))
    return codes, scales


def int4_matvec(x, codes, scales, group: int, zeros=None, x_scales=None, out_dtype=None, stream=None):
    """Products of a few rows with 4-bit weights: ``x @ ((u - zeros) * scales).T`` with a scale
    and a zero point (8 without ``zeros``) for each ``group`` of a weight row's columns.

    ``codes`` uint8 [out_dim, ceil(in_dim / 2)], two weights a byte, the even column's in the
    low half; ``scales`` [out_dim, ceil(in_dim / group)] float32, bfloat16 or float16; ``zeros``
    uint8 of that shape. ``x`` [rows, in_dim] float32, bfloat16 or float16, or the int8 or e4m3
    codes of :func:`add_rmsnorm_quant` with its scales as ``x_scales`` (one a row, or of the
    same ``group``). Returns [rows, out_dim] of ``out_dtype`` (``x``'s type; float32 for codes).
    Row pitches of ``codes`` that are multiples of 16 bytes are the fast ones."""
    import torch
    kind = _type_of(x.dtype)
    _need(kind is not None, "x must be float32, bfloat16, float16, int8 or float8_e4m3fn")
    _need(x.dim() == 2 and codes.dim() == 2, "x and codes must have two dimensions")
    rows, in_dim = x.shape
    out_dim = codes.shape[0]
    on = _On(x, stream)
    ldx = _pitch(x, "x", rows, in_dim, x.dtype, on.device)
    ldw = _pitch(codes, "codes", out_dim, (in_dim + 1) // 2, torch.uint8, on.device)
    _need(group >= 32 and group % 32 == 0, "group must be a multiple of 32")
    parts = -(-in_dim // group)
    scale_kind = _row_type(scales, "scales")
    _dense(scales, "scales", (out_dim, parts), scales.dtype, on.device)
    if zeros is not None:
        _dense(zeros, "zeros", (out_dim, parts), torch.uint8, on.device)
    _need((x_scales is not None) == (kind >= T_S8), "x_scales go with 8-bit rows, and only with them")
    x_group = 0
    if x_scales is not None:
        if x_scales.dim() == 2 and x_scales.shape[1] == parts and parts > 1:
            x_group = group
        _dense(x_scales, "x_scales", (rows, parts if x_group else 1), torch.float32, on.device)
    if out_dtype is None:
        out_dtype = x.dtype if kind <= T_F16 else torch.float32
    out = on.empty(rows, out_dim, dtype=out_dtype)
    on.run(lib().mmfree_cuda_int4_matvec, out.data_ptr(), x.data_ptr(), ldx, _ptr(x_scales),
           codes.data_ptr(), ldw, scales.data_ptr(), _ptr(zeros), rows, in_dim, out_dim, group, x_group,
           kind, scale_kind, _row_type(out, "out_dtype"), held=(x, codes, scales, zeros, x_scales))
    return out


def _sequences(on, rows: int, seq_starts, slots, state, step: bool) -> tuple[int, int]:
    """(sequences, states) of a call over packed rows, checked."""
    import torch
    if step:
        seqs = rows
    elif seq_starts is None:
        seqs = 1
    else:
        _need(seq_starts.dim() == 1 and seq_starts.shape[0] >= 1, "seq_starts must be [sequences + 1]")
        seqs = seq_starts.shape[0] - 1
        _dense(seq_starts, "seq_starts", (seqs + 1,), torch.int32, on.device)
    if slots is not None:
        _need(state is not None, "slots need a state")
        _dense(slots, "slots", (seqs,), torch.int32, on.device)
    count = seqs if state is None else state.shape[0]
    _need(slots is not None or count >= seqs, f"{count} states for {seqs} sequences")
    return seqs, count


def _causal_conv(x, weight, bias, state, seq_starts, slots, silu, out, stream, step):
    import torch
    kind = _row_type(x, "x")
    _need(x.dim() == 2 and weight.dim() == 2, "x and weight must have two dimensions")
    rows, channels = x.shape
    width = weight.shape[1]
    on = _On(x, stream)
    ldx = _pitch(x, "x", rows, channels, x.dtype, on.device)
    _need(2 <= width <= 8, "weight must be [channels, 2 to 8]")
    _dense(weight, "weight", (channels, width), torch.float32, on.device)
    if bias is not None:
        _dense(bias, "bias", (channels,), torch.float32, on.device)
    if state is not None:
        _need(state.dim() == 3, "state must be [states, width - 1, channels]")
        _dense(state, "state", (state.shape[0], width - 1, channels), x.dtype, on.device)
        _apart(state, "state", x, "x")
    seqs, count = _sequences(on, rows, seq_starts, slots, state, step)
    if out is None:
        out = on.empty(rows, channels, dtype=x.dtype)
    else:
        for t, name in ((x, "x"), (weight, "weight"), (bias, "bias"), (state, "state")):
            _apart(out, "out", t, name)
    a = ConvArgs(out.data_ptr(), x.data_ptr(), weight.data_ptr(), _ptr(bias), _ptr(state),
                 _ptr(seq_starts), _ptr(slots), _pitch(out, "out", rows, channels, x.dtype, on.device),
                 ldx, rows, seqs, count, channels, width, kind, int(silu))
    on.run(lib().mmfree_cuda_causal_conv_step if step else lib().mmfree_cuda_causal_conv, C.byref(a),
           held=(out, x, weight, bias, state, seq_starts, slots))
    return out


def causal_conv(x, weight, bias=None, state=None, seq_starts=None, slots=None, silu: bool = False,
                out=None, stream=None):
    """The short causal convolution of each channel along packed sequences: y[t] = bias + sum_j
    weight[:, j] * x[t - (width - 1) + j], through silu when asked for.

    ``x`` [tokens, channels] float32, bfloat16 or float16; ``weight`` float32 [channels, width],
    width 2 to 8, the newest input's tap last; ``bias`` float32 [channels]. ``seq_starts`` int32
    [sequences + 1] on the device: the first row of each sequence and the row behind the last
    (without: one sequence); rows outside the sequences are left as they were in ``out``.
    ``state`` [states, width - 1, channels] of ``x``'s type: the inputs before each sequence,
    oldest first, updated in place (without: zeros). ``slots`` int32 [sequences]: the state of
    each sequence (they must differ; a negative one marks a sequence that is left out).
    Starts or slots out of range are reported by :func:`kernel_status`."""
    return _causal_conv(x, weight, bias, state, seq_starts, slots, silu, out, stream, False)


def causal_conv_step(x, weight, state, bias=None, slots=None, silu: bool = False, out=None,
                     stream=None):
    """:func:`causal_conv` for one token of each stream: row s of ``x`` continues the sequence
    whose inputs are in state ``slots[s]`` (s without ``slots``)."""
    _need(state is not None, "a step needs a state")
    return _causal_conv(x, weight, bias, state, None, slots, silu, out, stream, True)


def _selective(x, dt, A, B, C_, D, z, dt_bias, dt_softplus, state, seq_starts, slots, out, stream,
               step):
    import torch
    kind = _row_type(x, "x")
    _need(x.dim() == 2 and A.dim() == 2, "x and A must have two dimensions")
    rows, channels = x.shape
    states = A.shape[1]
    on = _On(x, stream)
    dev = on.device
    ldx = _pitch(x, "x", rows, channels, x.dtype, dev)
    ld_dt = _pitch(dt, "dt", rows, channels, x.dtype, dev)
    ldz = 0 if z is None else _pitch(z, "z", rows, channels, x.dtype, dev)
    _need(1 <= states <= 256, "A must be [channels, 1 to 256]")
    _dense(A, "A", (channels, states), torch.float32, dev)
    groups = B.shape[1] if B.dim() == 3 else 1
    _need(groups >= 1 and channels % groups == 0, f"{groups} groups do not divide {channels} channels")

    def mixed(t, name):  # [rows, states] or [rows, groups, states]
        _need(t.device == dev, f"{name} is on {t.device}, not on {dev}")
        _need(t.dtype == x.dtype, f"{name} must be {x.dtype}, not {t.dtype}")
        _need(tuple(t.shape) == ((rows, groups, states) if B.dim() == 3 else (rows, states)),
              f"{name} must be [rows, states] or [rows, groups, states], not {list(t.shape)}")
        s = t.stride()
        _need((s[-1] == 1 or states == 1) and (groups == 1 or s[-2] == states),
              f"{name}'s rows must be contiguous")
        return s[0]

    ldb, ldc = mixed(B, "B"), mixed(C_, "C")
    if D is not None:
        _dense(D, "D", (channels,), torch.float32, dev)
    if dt_bias is not None:
        _dense(dt_bias, "dt_bias", (channels,), torch.float32, dev)
    if state is not None:
        _need(state.dim() == 3, "state must be [states, channels, A's columns]")
        _dense(state, "state", (state.shape[0], channels, states), torch.float32, dev)
        for t, name in ((x, "x"), (dt, "dt"), (A, "A"), (B, "B"), (C_, "C"), (z, "z")):
            _apart(state, "state", t, name)
    seqs, count = _sequences(on, rows, seq_starts, slots, state, step)
    if out is None:
        out = on.empty(rows, channels, dtype=x.dtype)
    else:
        for t, name in ((x, "x"), (dt, "dt"), (A, "A"), (B, "B"), (C_, "C"), (z, "z"), (D, "D"),
                        (dt_bias, "dt_bias"), (state, "state")):
            _apart(out, "out", t, name)
    a = SsmArgs(out.data_ptr(), x.data_ptr(), dt.data_ptr(), _ptr(z), B.data_ptr(), C_.data_ptr(),
                A.data_ptr(), _ptr(D), _ptr(dt_bias), _ptr(state), _ptr(seq_starts), _ptr(slots),
                _pitch(out, "out", rows, channels, x.dtype, dev), ldx, ld_dt, ldz, ldb, ldc, rows, seqs,
                count, channels, states, groups, kind, int(dt_softplus))
    on.run(lib().mmfree_cuda_selective_step if step else lib().mmfree_cuda_selective_scan, C.byref(a),
           held=(out, x, dt, z, B, C_, A, D, dt_bias, state, seq_starts, slots))
    return out


def selective_scan(x, dt, A, B, C, D=None, z=None, dt_bias=None, dt_softplus: bool = True,
                   state=None, seq_starts=None, slots=None, out=None, stream=None):
    """The selective state space scan along packed sequences. For each channel d, with delta =
    softplus(dt + dt_bias) (dt + dt_bias without ``dt_softplus``)::

        h[n] = exp(delta * A[d, n]) * h[n] + delta * x * B[n]
        y    = (sum_n C[n] * h[n] + D[d] * x) * z * sigmoid(z)

    ``x``, ``dt`` and ``z`` [tokens, channels], ``B`` and ``C`` [tokens, states] or [tokens,
    groups, states], all of one type (float32, bfloat16 or float16); ``A`` [channels, states],
    ``D`` and ``dt_bias`` [channels] and ``state`` [states, channels, A's columns] float32, the
    state updated in place (without: zeros). ``seq_starts``, ``slots`` and ``out`` as in
    :func:`causal_conv`. Returns y of ``x``'s type."""
    return _selective(x, dt, A, B, C, D, z, dt_bias, dt_softplus, state, seq_starts, slots, out, stream,
                      False)


def selective_step(x, dt, A, B, C, state, D=None, z=None, dt_bias=None, dt_softplus: bool = True,
                   slots=None, out=None, stream=None):
    """:func:`selective_scan` for one token of each stream: row s continues the sequence in
    state ``slots[s]`` (s without ``slots``)."""
    _need(state is not None, "a step needs a state")
    return _selective(x, dt, A, B, C, D, z, dt_bias, dt_softplus, state, None, slots, out, stream, True)
