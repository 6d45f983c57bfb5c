"""Tensor-level wrappers over the C ABI.

Each function validates its tensors the way the reference's native bridge
does (defined, on the device, exact dtype, contiguous:
acceleration/custom_ops/qwen2_5_vl/aclnn_grouped_swiglu_out_bridge.cpp:101-109),
allocates the outputs with the input's device, and launches on the current
CUDA stream.  torch is used for memory and streams only; all arithmetic is in
the CUDA library.  Nothing here falls back to torch math.
"""
from __future__ import annotations

import torch

from . import _lib

_err_words: dict[int, torch.Tensor] = {}
_index_words: dict[int, torch.Tensor] = {}


def _stream() -> int:
    return torch.cuda.current_stream().cuda_stream


def _req(t: torch.Tensor, name: str, dtype, ndim: int | None = None) -> torch.Tensor:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor (there is no CPU path)")
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if ndim is not None and t.dim() != ndim:
        raise ValueError(f"{name} must be {ndim}D, got shape {tuple(t.shape)}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    return t


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def _workspace(nbytes: int, device: torch.device, kind: str = "decode", own_in_capture: bool = False) -> torch.Tensor:
    """Zero-initialised scratch, one per (device, stream, kind) and, under capture, one per captured stream of the graph,
    grown on demand (``csrc/host_path.cpp`` keeps it).

    The decode kernels leave their part zeroed where it has to be, so it is
    cleared only when it is (re)allocated; the prefill and W8A8 split-K partial
    sums overwrite theirs freely, hence the separate kinds.  With ``own_in_capture``
    a graph capture may begin on a stream that has none; else that is an error.
    """
    index = device.index if device.index is not None else torch.cuda.current_device()
    return _lib.host().workspace(nbytes, index, kind, own_in_capture)


def new_workspace(nbytes: int, device) -> torch.Tensor:
    """A zero-filled scratch buffer for callers that manage scratch themselves (CUDA graphs)."""
    return torch.zeros(max(int(nbytes), 1 << 16), dtype=torch.uint8, device=device)


def w4a16_decode_workspace_bytes(m: int, n: int, k: int, k_split: int = 0) -> int:
    return int(_lib.load().mp_w4a16_decode_workspace_bytes_ex(m, n, k, k_split))


def w4a16_decode_kernel_choice(m: int, n: int, k: int, have_workspace: bool = True) -> str:
    """Name of the kernel the process default picks for a call of :func:`w4a16_linear_decode` of this shape
    (1 <= m <= 64); above 16 rows ``"mma_sync"`` means the split-K kernel.  :func:`w4a16_linear` has a rule of its own."""
    kind = _lib.load().mp_w4a16_decode_kernel_choice(m, n, k, 1 if have_workspace else 0)
    _lib.check(min(kind, 0), "w4a16_decode_kernel_choice", M=m, N=n, K=k)
    return {0: "mma_sync", 1: "umma"}[kind]


# ------------------------------------------------------------------ W4A16
def w4a16_quantize(weight: torch.Tensor, group_size: int = 128):
    """Asymmetric int4 group quantisation + packing of ``weight[N,K]`` (fp16).

    Returns ``(weight_packed int32[N,K/8], weight_scale f16[N,G],
    weight_zero_point int32[N,ceil(G/8)], group_size_used)``.  When ``K`` is
    not a multiple of ``group_size`` one group spans the row, as the
    reference does (quantizer.py:67-68).
    """
    w = _req(weight, "weight", torch.float16, 2)
    n, k = w.shape
    g = group_size if (group_size > 0 and k % group_size == 0) else k
    made = _lib.host().w4_quantize(w, g)
    if isinstance(made, int):
        _lib.check(made, "w4a16_quantize", N=n, K=k, group=g)
    packed, scale, zero = made
    return packed, scale, zero, g


def w4a16_dequant(weight_packed, weight_scale, weight_zero_point, out_features: int, in_features: int):
    """fp16 ``[N,K]`` weights ``f16((u - z) * s)``; ``weight_zero_point=None`` means z = 8."""
    p = _req(weight_packed, "weight_packed", torch.int32, 2)
    s = _req(weight_scale, "weight_scale", torch.float16, 2)
    z = None if weight_zero_point is None else _req(weight_zero_point, "weight_zero_point", torch.int32, 2)
    n, k = int(out_features), int(in_features)
    if p.shape != (n, k // 8) or k % 8:
        raise ValueError(f"weight_packed shape {tuple(p.shape)} does not match ({n}, {k}//8)")
    groups = s.shape[1]
    if s.shape[0] != n or k % groups:
        raise ValueError(f"weight_scale shape {tuple(s.shape)} does not divide K={k}")
    out = _lib.host().w4_dequant(p, s, z, n, k, k // groups)
    if isinstance(out, int):
        _lib.check(out, "w4a16_dequant", N=n, K=k, groups=groups)
    return out


def w4a16_prepare(weight_scale, weight_zero_point, in_features: int):
    """Group-major ``(scale, zero)`` fp16 pairs ``[G, N, 2]`` read by the GEMM kernels."""
    s = _req(weight_scale, "weight_scale", torch.float16, 2)
    z = None if weight_zero_point is None else _req(weight_zero_point, "weight_zero_point", torch.int32, 2)
    n, groups = s.shape
    k = int(in_features)
    sz = torch.empty((groups, n, 2), dtype=torch.float16, device=s.device)
    st = _lib.load().mp_w4a16_prepare(s.data_ptr(), _ptr(z), n, k, k // groups, sz.data_ptr(), _stream())
    _lib.check(st, "w4a16_prepare", N=n, K=k, groups=groups)
    return sz


_DECODE_OPT_KERNEL = {"mma_sync": 0x1, "umma": 0x2, "auto": 0x4}


def decode_options(kernel: str | None = None, pdl: bool | None = None) -> int:
    """The ``options`` word of ``mp_w4a16_linear_decode_opts``: kernel and programmatic dependent launch
    chosen for one call; ``None`` keeps the process default."""
    opt = 0
    if kernel is not None:
        if kernel not in _DECODE_OPT_KERNEL:
            raise ValueError(f"unknown decode kernel {kernel!r}; expected one of {sorted(_DECODE_OPT_KERNEL)}")
        opt |= _DECODE_OPT_KERNEL[kernel]
    if pdl is not None:
        opt |= 0x10 if pdl else 0x20
    return opt


def w4a16_linear_decode(x, weight_packed, scale_zero, bias=None, *, k_split: int = 0, workspace=None, out=None,
                        options: int = 0):
    """``y[M,N] = x[M,K] @ dequant(W)^T (+bias)`` with the weight-streaming kernels (M <= 64), for callers who choose
    kernel, split or scratch themselves; :func:`w4a16_linear` picks the fastest kernel for the shape.

    ``workspace`` (uint8, zero-filled when created, not shared by calls that
    may overlap) defaults to a cached buffer per device and stream.  ``options``
    (see :func:`decode_options`) fixes kernel / launch mode for this call; with 17..64 rows ``kernel="umma"``
    runs the tcgen05 kernel with a 32- or 64-token activation tile, the other choices the split-K kernel.
    """
    x2 = _req(x, "x", torch.float16, 2)
    p = _req(weight_packed, "weight_packed", torch.int32, 2)
    sz = _req(scale_zero, "scale_zero", torch.float16, 3)
    b = None if bias is None else _req(bias, "bias", torch.float16, 1)
    m, k = x2.shape
    n = p.shape[0]
    groups = sz.shape[0]
    if p.shape[1] * 8 != k or sz.shape[1] != n or k % groups:
        raise ValueError(f"shape mismatch: x{tuple(x2.shape)} packed{tuple(p.shape)} sz{tuple(sz.shape)}")
    lib = _lib.load()
    nbytes = lib.mp_w4a16_decode_workspace_bytes_ex(m, n, k, k_split)
    if workspace is not None:
        ws = _req(workspace, "workspace", torch.uint8, 1)
    else:
        ws = _workspace(nbytes, x2.device) if nbytes else None      # M <= 16 needs no scratch
    y = torch.empty((m, n), dtype=torch.float16, device=x2.device) if out is None else _req(out, "out", torch.float16, 2)
    if y.shape != (m, n):
        raise ValueError(f"out must be [{m}, {n}]")
    if options:
        if k_split:
            raise ValueError("options and k_split cannot be combined")
        st = lib.mp_w4a16_linear_decode_opts(x2.data_ptr(), p.data_ptr(), sz.data_ptr(), _ptr(b), y.data_ptr(),
                                             m, n, k, k // groups, _ptr(ws), 0 if ws is None else ws.numel(),
                                             int(options), _stream())
    else:
        st = lib.mp_w4a16_linear_decode_ex(x2.data_ptr(), p.data_ptr(), sz.data_ptr(), _ptr(b), y.data_ptr(),
                                           m, n, k, k // groups, _ptr(ws), 0 if ws is None else ws.numel(), k_split,
                                           _stream())
    _lib.check(st, "w4a16_linear_decode", M=m, N=n, K=k, group=k // groups)
    return y


def w4a16_linear_decode_host(x_host, weight_packed, scale_zero, bias=None, *, y_host=None, x_stage=None, y_stage=None,
                             workspace=None):
    """Decode linear (M <= 16) on HOST activations: H2D copy, kernel and D2H copy are enqueued on the
    current stream and the call returns without waiting; ``y_host`` is valid after the stream (or
    device) has been synchronised.  ``x_host`` / ``y_host`` are CPU fp16 tensors (pinned memory makes
    the copies asynchronous); ``x_stage`` / ``y_stage`` are optional device staging buffers to reuse;
    ``workspace`` (``new_workspace(w4a16_decode_workspace_bytes(m, n, k))``, not shared with calls that may
    overlap this one) lets the library pick among all decode kernels instead of the scratch-free ones.
    """
    if x_host.device.type != "cpu" or x_host.dtype != torch.float16 or x_host.dim() != 2 or not x_host.is_contiguous():
        raise ValueError("x_host must be a contiguous 2-D fp16 CPU tensor")
    p = _req(weight_packed, "weight_packed", torch.int32, 2)
    sz = _req(scale_zero, "scale_zero", torch.float16, 3)
    b = None if bias is None else _req(bias, "bias", torch.float16, 1)
    m, k = x_host.shape
    n = p.shape[0]
    groups = sz.shape[0]
    if p.shape[1] * 8 != k or sz.shape[1] != n or k % groups:
        raise ValueError(f"shape mismatch: x{tuple(x_host.shape)} packed{tuple(p.shape)} sz{tuple(sz.shape)}")
    if y_host is None:
        y_host = torch.empty((m, n), dtype=torch.float16).pin_memory()
    if y_host.device.type != "cpu" or y_host.dtype != torch.float16 or tuple(y_host.shape) != (m, n) \
            or not y_host.is_contiguous():
        raise ValueError(f"y_host must be a contiguous fp16 CPU tensor [{m}, {n}]")
    xs = torch.empty((m, k), dtype=torch.float16, device=p.device) if x_stage is None else _req(x_stage, "x_stage", torch.float16, 2)
    ys = torch.empty((m, n), dtype=torch.float16, device=p.device) if y_stage is None else _req(y_stage, "y_stage", torch.float16, 2)
    if tuple(xs.shape) != (m, k) or tuple(ys.shape) != (m, n):
        raise ValueError("staging buffers must be [M, K] and [M, N]")
    if workspace is not None and (not workspace.is_cuda or workspace.dtype != torch.uint8 or
                                  workspace.numel() < w4a16_decode_workspace_bytes(m, n, k)):
        raise ValueError("workspace must be a CUDA uint8 tensor of at least w4a16_decode_workspace_bytes(m, n, k) bytes")
    st = _lib.load().mp_w4a16_linear_decode_host_ws(
        x_host.data_ptr(), xs.data_ptr(), p.data_ptr(), sz.data_ptr(), _ptr(b), ys.data_ptr(), y_host.data_ptr(), m, n, k,
        k // groups, _ptr(workspace), 0 if workspace is None else workspace.numel(), _stream())
    _lib.check(st, "w4a16_linear_decode_host", M=m, N=n, K=k, group=k // groups)
    return y_host


def w4a16_linear_decode_static(x, weight_packed, scale_zero, bias=None, out=None):
    """Decode linear that takes no scratch from the caller and allocates none.

    For hosts that cannot allocate device memory (a plugin inside another
    runtime's forward pass, code running where ``cudaMalloc`` is off limits):
    the split-K scratch is a fixed 8 MiB array inside the library.  Pass
    ``out`` to keep this wrapper allocation-free as well.  Shapes whose
    partial sums exceed the array raise (status "workspace"); calls that may
    overlap on one device share the array and would race.
    """
    x2 = _req(x, "x", torch.float16, 2)
    p = _req(weight_packed, "weight_packed", torch.int32, 2)
    sz = _req(scale_zero, "scale_zero", torch.float16, 3)
    b = None if bias is None else _req(bias, "bias", torch.float16, 1)
    m, k = x2.shape
    n = p.shape[0]
    groups = sz.shape[0]
    if p.shape[1] * 8 != k or sz.shape[1] != n or k % groups:
        raise ValueError(f"shape mismatch: x{tuple(x2.shape)} packed{tuple(p.shape)} sz{tuple(sz.shape)}")
    y = torch.empty((m, n), dtype=torch.float16, device=x2.device) if out is None else _req(out, "out", torch.float16, 2)
    if y.shape != (m, n):
        raise ValueError(f"out must be [{m}, {n}]")
    st = _lib.load().mp_w4a16_linear_decode_static(x2.data_ptr(), p.data_ptr(), sz.data_ptr(), _ptr(b), y.data_ptr(),
                                                   m, n, k, k // groups, _stream())
    _lib.check(st, "w4a16_linear_decode_static", M=m, N=n, K=k, group=k // groups)
    return y


def w4a16_linear_prefill(x, weight_packed, scale_zero, bias=None, *, workspace=None):
    """``y = x @ dequant(W)^T (+bias)`` on the fp16 tensor cores with the dequant fused in.

    Shapes with few output tiles (M <= 256, narrow N) split K and need scratch: ``workspace`` (uint8)
    defaults to the cached per-(device, stream) buffer.
    """
    x2 = _req(x, "x", torch.float16, 2)
    p = _req(weight_packed, "weight_packed", torch.int32, 2)
    sz = _req(scale_zero, "scale_zero", torch.float16, 3)
    b = None if bias is None else _req(bias, "bias", torch.float16, 1)
    m, k = x2.shape
    n = p.shape[0]
    groups = sz.shape[0]
    if p.shape[1] * 8 != k or sz.shape[1] != n or k % groups:
        raise ValueError(f"shape mismatch: x{tuple(x2.shape)} packed{tuple(p.shape)} sz{tuple(sz.shape)}")
    y = torch.empty((m, n), dtype=torch.float16, device=x2.device)
    if m == 0:
        return y
    lib = _lib.load()
    nbytes = lib.mp_w4a16_prefill_workspace_bytes(m, n, k)
    if workspace is not None:
        ws = _req(workspace, "workspace", torch.uint8, 1)
    else:
        ws = _workspace(nbytes, x2.device, "prefill") if nbytes else None
    st = lib.mp_w4a16_linear_prefill_ex(x2.data_ptr(), p.data_ptr(), sz.data_ptr(), _ptr(b), y.data_ptr(),
                                        m, n, k, k // groups, _ptr(ws), 0 if ws is None else ws.numel(),
                                        _error_word(x2.device).data_ptr(), _stream())
    _lib.check(st, "w4a16_linear_prefill", M=m, N=n, K=k, group=k // groups)
    return y


def w4a16_linear(x, weight_packed, scale_zero, bias=None):
    """W4A16 linear for any number of rows: the library picks among the decode kernels, the tcgen05 weight-streaming
    kernel (up to 128 rows) and the tensor-core prefill kernel (``mp_w4a16_linear``).  Shapes the prefill kernel does
    not take (K or the group size not a multiple of 64) are processed by the decode kernels in 64-row slabs.
    """
    x2 = _req(x, "x", torch.float16, 2)
    p = _req(weight_packed, "weight_packed", torch.int32, 2)
    sz = _req(scale_zero, "scale_zero", torch.float16, 3)
    b = None if bias is None else _req(bias, "bias", torch.float16, 1)
    m, k = x2.shape
    n = p.shape[0]
    groups = sz.shape[0]
    if p.shape[1] * 8 != k or sz.shape[1] != n or k % groups:
        raise ValueError(f"shape mismatch: x{tuple(x2.shape)} packed{tuple(p.shape)} sz{tuple(sz.shape)}")
    group = k // groups
    if m == 0:
        return torch.empty((m, n), dtype=torch.float16, device=x2.device)
    if m > 16 and (k % 64 or group % 64):
        outs = [w4a16_linear_decode(x2[i:i + 64], p, sz, b) for i in range(0, m, 64)]
        return outs[0] if len(outs) == 1 else torch.cat(outs, dim=0)
    y = torch.empty((m, n), dtype=torch.float16, device=x2.device)
    lib = _lib.load()
    nbytes = lib.mp_w4a16_linear_workspace_bytes(m, n, k, group)
    ws = _workspace(nbytes, x2.device, own_in_capture=True) if nbytes else None
    st = lib.mp_w4a16_linear(x2.data_ptr(), p.data_ptr(), sz.data_ptr(), _ptr(b), y.data_ptr(), m, n, k, group, _ptr(ws),
                             0 if ws is None else ws.numel(), _error_word(x2.device).data_ptr(), _stream())
    _lib.check(st, "w4a16_linear", M=m, N=n, K=k, group=group)
    return y


# ------------------------------------------------------------------- W8A8
def act_quant_per_token(x, *, want_codes: bool = True, want_fake: bool = False):
    """Per-row symmetric int8 quantisation of ``x[..., K]`` (fp16).

    Returns ``(codes int8[...,K] | None, scale f32[...] | None, fake f16 | None)``.
    """
    xt = _req(x, "x", torch.float16)
    k = xt.shape[-1]
    m = xt.numel() // k
    q = torch.empty(xt.shape, dtype=torch.int8, device=xt.device) if want_codes else None
    s = torch.empty(xt.shape[:-1], dtype=torch.float32, device=xt.device) if want_codes else None
    f = torch.empty_like(xt) if want_fake else None
    if m == 0:
        return q, s, f
    st = _lib.load().mp_act_quant_per_token(xt.data_ptr(), m, k, _ptr(q), _ptr(s), _ptr(f), _stream())
    _lib.check(st, "act_quant_per_token", M=m, K=k)
    return q, s, f


_DECODE_KERNELS = {"mma_sync": 0, "umma": 1, "auto": 2}


def set_decode_kernel(kind: str) -> str:
    """Choose the kernel behind the W4A16 linears of few rows; returns the previous choice.

    ``"umma"``: tcgen05.mma with the dequantised weights as the tensor-memory operand;
    ``"mma_sync"``: the mma.sync kernels; ``"auto"`` (the default): by shape.  Shapes the
    chosen kernel does not take fall through to the other ones.  This is the process-wide default;
    a single call chooses with ``options=decode_options(kernel=...)``.
    """
    if kind not in _DECODE_KERNELS:
        raise ValueError(f"unknown decode kernel {kind!r}; expected one of {sorted(_DECODE_KERNELS)}")
    prev = _lib.load().mp_set_decode_kernel(_DECODE_KERNELS[kind])
    if prev < 0:
        _lib.check(prev, "set_decode_kernel", kind=kind)
    return next(k for k, v in _DECODE_KERNELS.items() if v == prev)


def _error_word(device: torch.device) -> torch.Tensor:
    """Per-device int32 the tensor-core kernels set when a bounded wait gives up."""
    idx = device.index if device.index is not None else torch.cuda.current_device()
    w = _err_words.get(idx)
    if w is None:
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("first use of a tensor-core op must happen outside CUDA graph capture")
        w = torch.zeros(1, dtype=torch.int32, device=device)
        _err_words[idx] = w
    return w


def _index_word(device: torch.device) -> int:
    """Address of the per-device int32 the attention kernels set when an index they read is out of range."""
    idx = device.index if device.index is not None else torch.cuda.current_device()
    w = _index_words.get(idx)
    if w is None:
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("first use of an attention op must happen outside CUDA graph capture")
        w = torch.zeros(1, dtype=torch.int32, device=device)
        _index_words[idx] = w
    return w.data_ptr()


def check_device_errors(device=None) -> None:
    """Synchronise and raise if any kernel reported a device-side wait that gave up, or an attention kernel an index
    (position, slot, page, length, sequence end) that was out of range.

    A kernel that gave up leaves its arrival counters and partial sums as they were at that moment, so the
    scratch buffers this module caches are cleared again before the error is raised and later calls start from
    a clean state.  Scratch owned by the caller (``new_workspace``) must be zeroed by the caller, and the
    tensor- and expert-parallel modules, whose call numbers and arrival words are spread over the ranks, must
    be rebuilt on every rank after such an error."""
    torch.cuda.synchronize(device)
    import ctypes

    def rearm(index=None):
        for dev_index, ws in _lib.host().workspaces():
            if index is None or dev_index == index:
                ws.zero_()
        torch.cuda.synchronize(device)

    flag = ctypes.c_int(0)
    _lib.check(_lib.load().mp_read_decode_error(ctypes.byref(flag)), "read_decode_error")
    if flag.value != 0:
        rearm()
        raise _lib.MindPipeKernelError("a bounded wait inside a decode kernel timed out")
    for idx, w in _err_words.items():
        if int(w.item()) != 0:
            w.zero_()
            rearm(idx)
            raise _lib.MindPipeKernelError(f"device {idx}: a bounded wait inside a tensor-core kernel timed out")
    for idx, w in _index_words.items():
        if int(w.item()) != 0:
            w.zero_()
            raise _lib.MindPipeKernelError(f"device {idx}: an attention call was given a position, slot, page, length or "
                                           "sequence end out of range")


def w8a8_gemm(qx, x_scale, weight_i8, weight_scale, bias=None, *, workspace=None):
    """``f16((qx @ w^T) * x_scale[:,None] * w_scale[None,:] (+bias))`` with int32 accumulation.

    At decode / small-batch row counts K is split over the SMs (bit-identical result); the scratch for
    that is ``workspace`` (uint8) or the cached per-(device, stream) buffer.
    """
    a = _req(qx, "qx", torch.int8, 2)
    b = _req(weight_i8, "weight", torch.int8, 2)
    sa = _req(x_scale, "x_scale", torch.float32, 1)
    sb = _req(weight_scale, "weight_scale", torch.float32, 1)
    bi = None if bias is None else _req(bias, "bias", torch.float16, 1)
    m, k = a.shape
    n = b.shape[0]
    if b.shape[1] != k or sa.numel() != m or sb.numel() != n:
        raise ValueError(f"shape mismatch: qx{tuple(a.shape)} w{tuple(b.shape)} sx{tuple(sa.shape)} sw{tuple(sb.shape)}")
    y = torch.empty((m, n), dtype=torch.float16, device=a.device)
    if m == 0:
        return y
    lib = _lib.load()
    nbytes = lib.mp_w8a8_gemm_workspace_bytes(m, n, k)
    if workspace is not None:
        ws = _req(workspace, "workspace", torch.uint8, 1)
    else:
        ws = _workspace(nbytes, a.device, "w8a8") if nbytes else None
    st = lib.mp_w8a8_gemm_ex(a.data_ptr(), sa.data_ptr(), b.data_ptr(), sb.data_ptr(), _ptr(bi), y.data_ptr(),
                             m, n, k, _ptr(ws), 0 if ws is None else ws.numel(), _error_word(a.device).data_ptr(),
                             _stream())
    _lib.check(st, "w8a8_gemm", M=m, N=n, K=k)
    return y


def w8a8_gemm_i32(qx, weight_i8):
    """Raw int32 accumulators ``qx @ w^T``."""
    a = _req(qx, "qx", torch.int8, 2)
    b = _req(weight_i8, "weight", torch.int8, 2)
    m, k = a.shape
    n = b.shape[0]
    if b.shape[1] != k:
        raise ValueError(f"shape mismatch: qx{tuple(a.shape)} w{tuple(b.shape)}")
    acc = torch.empty((m, n), dtype=torch.int32, device=a.device)
    if m == 0:
        return acc
    st = _lib.load().mp_w8a8_gemm_i32(a.data_ptr(), b.data_ptr(), acc.data_ptr(), m, n, k,
                                      _error_word(a.device).data_ptr(), _stream())
    _lib.check(st, "w8a8_gemm_i32", M=m, N=n, K=k)
    return acc


# -------------------------------------------------------------------- MoE
def moe_router_topk(logits, top_k: int = 2):
    """softmax(fp32) -> top-k -> renormalise -> fp16.  Returns ``(index int32[T,k], weights f16[T,k])``."""
    lg = _req(logits, "logits", torch.float32, 2)
    t, e = lg.shape
    idx = torch.empty((t, top_k), dtype=torch.int32, device=lg.device)
    w = torch.empty((t, top_k), dtype=torch.float16, device=lg.device)
    if t:
        st = _lib.load().mp_moe_router_topk(lg.data_ptr(), t, e, top_k, idx.data_ptr(), w.data_ptr(), _stream())
        _lib.check(st, "moe_router_topk", T=t, E=e, k=top_k)
    return idx, w


class MoeRouting:
    """Device-side result of routing + gather + quant for the experts one GPU owns."""

    __slots__ = ("plan", "dest_row", "routed_q", "routed_scale", "padded_rows", "num_local_experts")

    def __init__(self, plan, dest_row, routed_q, routed_scale, padded_rows, num_local_experts):
        self.plan, self.dest_row, self.routed_q, self.routed_scale = plan, dest_row, routed_q, routed_scale
        self.padded_rows, self.num_local_experts = padded_rows, num_local_experts

    @property
    def counts(self):
        return self.plan[: self.num_local_experts]

    @property
    def segment_offsets(self):
        e = self.num_local_experts
        return self.plan[2 * e: 3 * e + 1]


def moe_route_gather_quant(hidden, top_k_index, expert_lo: int, expert_hi: int, out=None) -> MoeRouting:
    """Sort the routed rows of experts ``[expert_lo, expert_hi)`` by expert and quantise them per token.

    ``out = (plan, routed_q, routed_scale)`` writes into caller buffers (e.g. symmetric memory)."""
    hs = _req(hidden, "hidden_states", torch.float16, 2)
    ids = _req(top_k_index, "top_k_index", torch.int32, 2)
    t, h = hs.shape
    k = ids.shape[1]
    if ids.shape[0] != t:
        raise ValueError("top_k_index and hidden_states disagree on the number of tokens")
    e = expert_hi - expert_lo
    lib = _lib.load()
    padded = lib.mp_moe_padded_rows(e, t * k)
    dest = torch.empty(t * k, dtype=torch.int32, device=hs.device)
    if out is None:
        plan = torch.empty(lib.mp_moe_plan_ints(e, t * k), dtype=torch.int32, device=hs.device)
        rq = torch.empty((padded, h), dtype=torch.int8, device=hs.device)
        rs = torch.empty(padded, dtype=torch.float32, device=hs.device)
    else:
        plan, rq, rs = out
        if plan.numel() < lib.mp_moe_plan_ints(e, t * k) or rq.shape[0] < padded or rs.numel() < padded:
            raise ValueError("routing buffers are too small for this many tokens")
    st = lib.mp_moe_route_gather_quant(hs.data_ptr(), ids.data_ptr(), t, h, k, expert_lo, expert_hi, plan.data_ptr(),
                                       dest.data_ptr(), rq.data_ptr(), rs.data_ptr(), _stream())
    _lib.check(st, "moe_route_gather_quant", T=t, H=h, k=k, experts=(expert_lo, expert_hi))
    return MoeRouting(plan, dest, rq, rs, padded, e)


def moe_expert_stage(routed_q, routed_scale, plan, num_local_experts: int, w13_q, w13_scale, w2_q, w2_scale):
    """Grouped GEMM1 + SwiGLU + re-quant + grouped GEMM2 on expert-sorted int8 rows -> f16 ``[padded_rows, H]``."""
    rq = _req(routed_q, "routed_q", torch.int8, 2)
    rs = _req(routed_scale, "routed_scale", torch.float32, 1)
    pl = _req(plan, "plan", torch.int32, 1)
    w13 = _req(w13_q, "w13", torch.int8, 3)
    s13 = _req(w13_scale, "w13_scale", torch.float32, 2)
    w2 = _req(w2_q, "w2", torch.int8, 3)
    s2 = _req(w2_scale, "w2_scale", torch.float32, 2)
    padded, h = rq.shape
    e, two_i, h2 = w13.shape
    i = two_i // 2
    if e != num_local_experts or h2 != h or tuple(w2.shape) != (e, h, i) or tuple(s13.shape) != (e, two_i) or \
            tuple(s2.shape) != (e, h) or rs.numel() != padded:
        raise ValueError("expert weight / routed buffer shapes are inconsistent")
    lib = _lib.load()
    nbytes = lib.mp_moe_expert_stage_workspace_bytes(padded, i)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=rq.device)      # served by torch's caching allocator
    d = torch.empty((padded, h), dtype=torch.float16, device=rq.device)
    st = lib.mp_moe_expert_stage(rq.data_ptr(), rs.data_ptr(), pl.data_ptr(), padded, h, i, e, w13.data_ptr(),
                                 s13.data_ptr(), w2.data_ptr(), s2.data_ptr(), d.data_ptr(), ws.data_ptr(), nbytes,
                                 _error_word(rq.device).data_ptr(), _stream())
    _lib.check(st, "moe_expert_stage", padded_rows=padded, H=h, I=i, E=e)
    return d


def w8a8_gate_up_swiglu_requant(x_q, x_scale, w_q, w_scale):
    """Chunked gate/up projection + SwiGLU + per-token re-quant on int8 rows, all chunks in one grouped launch.

    ``x_q`` int8 ``[T, H]``, ``x_scale`` fp32 ``[T]``, ``w_q`` int8 ``[chunks, 2C, H]`` (per chunk: gate rows, then up
    rows), ``w_scale`` fp32 ``[chunks, 2C]`` -> (int8 ``[chunks, T, C]``, fp32 ``[chunks, T]``)."""
    xq = _req(x_q, "x", torch.int8, 2)
    xs = _req(x_scale, "x_scale", torch.float32, 1)
    w = _req(w_q, "weight", torch.int8, 3)
    s = _req(w_scale, "weight_scale", torch.float32, 2)
    t, h = xq.shape
    chunks, two_c, h2 = w.shape
    c = two_c // 2
    if h2 != h or two_c % 2 or tuple(s.shape) != (chunks, two_c) or xs.numel() != t:
        raise ValueError("gate/up weight, scale and activation shapes are inconsistent")
    q = torch.empty((chunks, t, c), dtype=torch.int8, device=xq.device)
    qs = torch.empty((chunks, t), dtype=torch.float32, device=xq.device)
    if t == 0:
        return q, qs
    lib = _lib.load()
    nbytes = lib.mp_w8a8_gate_up_swiglu_requant_workspace_bytes(t, h, c, chunks)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=xq.device)
    st = lib.mp_w8a8_gate_up_swiglu_requant(xq.data_ptr(), xs.data_ptr(), w.data_ptr(), s.data_ptr(), t, h, c, chunks,
                                            q.data_ptr(), qs.data_ptr(), ws.data_ptr(), nbytes,
                                            _error_word(xq.device).data_ptr(), _stream())
    _lib.check(st, "w8a8_gate_up_swiglu_requant", T=t, H=h, C=c, chunks=chunks)
    return q, qs


_LOOP_OUT_WEIGHTS: dict = {}


def loop_out_weights(batched_weight, batched_weight_scale):
    """The reference's ``[chunks, H, 2C]`` gate/up weight and ``[chunks, 2C]`` scale in the layout the kernel
    streams (``[chunks, 2C, H]``, fp32 scales).  Made once per weight tensor and kept: weights are static while
    serving (the cache is keyed by storage address and version, so an in-place update makes a new copy)."""
    key = (batched_weight.data_ptr(), batched_weight._version, batched_weight_scale.data_ptr(),
           batched_weight_scale._version, tuple(batched_weight.shape))
    hit = _LOOP_OUT_WEIGHTS.get(key)
    if hit is None:
        if batched_weight.dtype != torch.int8 or batched_weight.dim() != 3:
            raise ValueError("batched_weight must be int8 [chunks, H, 2C]")
        chunks = batched_weight.shape[0]
        w = batched_weight.transpose(1, 2).contiguous()
        s = batched_weight_scale.reshape(chunks, -1).to(torch.float32).contiguous()
        _LOOP_OUT_WEIGHTS.clear()                       # one layer set resident per call site is the common case
        hit = _LOOP_OUT_WEIGHTS[key] = (w, s)
    return hit


def grouped_swiglu_loop_out(x, weights, batched_weight, group_list, weight_scales, batched_weight_scale, x_scale,
                            min_tokens: int = 0, layer_idx: int = -1):
    """The reference's loop-out op with its argument list (acceleration/runtime_patches/vllm.patch:114-170):
    ``x`` int8 ``[T, H]``; ``weights`` the per-chunk ``[1, H, 2C]`` views of ``batched_weight``
    ``[chunks, H, 2C]``; ``group_list`` int64 ``[1]`` (= T); ``weight_scales`` the per-chunk ``[1, 2C]`` views of
    ``batched_weight_scale``; ``x_scale`` fp32 ``[T]``.  Returns (int8 ``[chunks, T, C]``, fp32 ``[chunks, T]``).
    The reference switches between a per-chunk loop and one batched call at ``min_tokens``; here every size
    takes the single grouped launch, so ``min_tokens`` and ``layer_idx`` (a logging tag) only keep the
    signature.  Argument checks as the bridge's (aclnn_grouped_swiglu_out_bridge.cpp:166-199)."""
    if not weights or len(weights) != len(weight_scales):
        raise RuntimeError("loop-out requires equal non-empty weight lists")
    chunks = len(weights)
    if batched_weight.shape[0] != chunks or batched_weight_scale.shape[0] != chunks:
        raise RuntimeError("loop-out batched weight has an invalid chunk count")
    if x.dim() != 2 or x.dtype != torch.int8:
        raise RuntimeError("x must be a 2-D int8 tensor")
    if x_scale.dim() != 1 or x_scale.shape[0] != x.shape[0]:
        raise RuntimeError("x_scale must be [tokens]")
    if group_list.dim() != 1 or group_list.numel() != 1 or group_list.dtype != torch.int64:
        raise RuntimeError("group_list must be int64 [1]")
    width = batched_weight_scale.shape[-1]
    for wv, sv in zip(weights, weight_scales):
        if wv.shape[-1] != width or sv.shape[-1] != width or wv.shape[-2] != x.shape[1]:
            raise RuntimeError("loop-out weight view shapes differ")
    w, s = loop_out_weights(batched_weight, batched_weight_scale)
    return w8a8_gate_up_swiglu_requant(x.contiguous(), x_scale.to(torch.float32).contiguous(), w, s)


def moe_combine(d, dest_row, top_k_index, top_k_weights, num_tokens: int):
    """``out[t] = sum_j f16(d[dest(t,j)] * w[t,j])`` (fp16 adds, experts ascending)."""
    dd = _req(d, "d", torch.float16, 2)
    dr = _req(dest_row, "dest_row", torch.int32, 1)
    ids = _req(top_k_index, "top_k_index", torch.int32, 2)
    w = _req(top_k_weights, "top_k_weights", torch.float16, 2)
    k = ids.shape[1]
    h = dd.shape[1]
    out = torch.empty((num_tokens, h), dtype=torch.float16, device=dd.device)
    if num_tokens:
        st = _lib.load().mp_moe_combine(dd.data_ptr(), dr.data_ptr(), ids.data_ptr(), w.data_ptr(), num_tokens, h, k,
                                        out.data_ptr(), _stream())
        _lib.check(st, "moe_combine", T=num_tokens, H=h, k=k)
    return out


def gather_rows(src, row_map, out=None):
    """``dst[i] = src[row_map[i]]`` for a 1-D or 2-D ``src``; negative map entries give zero rows."""
    m = _req(row_map, "row_map", torch.int32, 1)
    if not src.is_cuda or not src.is_contiguous():
        raise ValueError("src must be a contiguous CUDA tensor")
    row_bytes = src.element_size() * (src.shape[1] if src.dim() == 2 else 1)
    shape = (m.numel(),) + tuple(src.shape[1:])
    dst = torch.empty(shape, dtype=src.dtype, device=src.device) if out is None else out
    if m.numel():
        st = _lib.load().mp_gather_rows(src.data_ptr(), m.data_ptr(), m.numel(), row_bytes, dst.data_ptr(), _stream())
        _lib.check(st, "gather_rows", rows=m.numel(), row_bytes=row_bytes)
    return dst


def add_rmsnorm_quant(x, residual, gamma, eps: float = 1e-5):
    """``residual += x`` (fp16), RMSNorm with ``gamma``, per-token int8 quant.

    Returns ``(codes int8[...,H], scale f32[...])`` -- the tuple input of the W8A8
    linear -- and updates ``residual`` in place.
    """
    xt = _req(x, "x", torch.float16)
    rt = _req(residual, "residual", torch.float16)
    g = _req(gamma, "gamma", torch.float16, 1)
    h = xt.shape[-1]
    if rt.shape != xt.shape or g.numel() != h:
        raise ValueError("x, residual and gamma shapes disagree")
    m = xt.numel() // h
    q = torch.empty(xt.shape, dtype=torch.int8, device=xt.device)
    s = torch.empty(xt.shape[:-1], dtype=torch.float32, device=xt.device)
    if m:
        st = _lib.load().mp_add_rmsnorm_quant(xt.data_ptr(), rt.data_ptr(), g.data_ptr(), float(eps), m, h, q.data_ptr(),
                                              s.data_ptr(), _stream())
        _lib.check(st, "add_rmsnorm_quant", M=m, H=h)
    return q, s


def affine_quant_per_row(x, *, want_fake: bool = False):
    """OmniQuant-style dynamic asymmetric 8-bit quantisation of each row of ``x[..., K]`` (fp16).

    Returns ``(codes uint8, scale f32, zero_point f32, rowsum int32, fake f16 | None)``.
    """
    xt = _req(x, "x", torch.float16)
    k = xt.shape[-1]
    m = xt.numel() // k
    q = torch.empty(xt.shape, dtype=torch.uint8, device=xt.device)
    s = torch.empty(xt.shape[:-1], dtype=torch.float32, device=xt.device)
    z = torch.empty(xt.shape[:-1], dtype=torch.float32, device=xt.device)
    rs = torch.empty(xt.shape[:-1], dtype=torch.int32, device=xt.device)
    f = torch.empty_like(xt) if want_fake else None
    if m:
        st = _lib.load().mp_affine_quant_per_row(xt.data_ptr(), m, k, q.data_ptr(), s.data_ptr(), z.data_ptr(),
                                                 rs.data_ptr(), _ptr(f), _stream())
        _lib.check(st, "affine_quant_per_row", M=m, K=k)
    return q, s, z, rs, f


def w8a8_affine_gemm(qx, x_scale, x_zero, x_rowsum, weight_u8, weight_scale, weight_zero, weight_rowsum, bias=None):
    """``f16(sum_k (qx - zx)(qw - zw) * sx * sw (+bias))`` from unsigned 8-bit codes."""
    a = _req(qx, "qx", torch.uint8, 2)
    b = _req(weight_u8, "weight", torch.uint8, 2)
    args = [_req(x_scale, "x_scale", torch.float32, 1), _req(x_zero, "x_zero", torch.float32, 1),
            _req(x_rowsum, "x_rowsum", torch.int32, 1), _req(weight_scale, "weight_scale", torch.float32, 1),
            _req(weight_zero, "weight_zero", torch.float32, 1), _req(weight_rowsum, "weight_rowsum", torch.int32, 1)]
    bi = None if bias is None else _req(bias, "bias", torch.float16, 1)
    m, k = a.shape
    n = b.shape[0]
    if b.shape[1] != k or any(t.numel() != m for t in args[:3]) or any(t.numel() != n for t in args[3:]):
        raise ValueError("shape mismatch between codes and their per-row parameters")
    y = torch.empty((m, n), dtype=torch.float16, device=a.device)
    if m == 0:
        return y
    st = _lib.load().mp_w8a8_affine_gemm(a.data_ptr(), args[0].data_ptr(), args[1].data_ptr(), args[2].data_ptr(),
                                         b.data_ptr(), args[3].data_ptr(), args[4].data_ptr(), args[5].data_ptr(),
                                         _ptr(bi), y.data_ptr(), m, n, k, _error_word(a.device).data_ptr(), _stream())
    _lib.check(st, "w8a8_affine_gemm", M=m, N=n, K=k)
    return y


# -------------------------------------------------------------- attention
def _on_gpu(t, name):
    """The checks that need no library, so that a machine without a GPU gives the same errors."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor (there is no CPU path)")
    return t.device


def rotary_append_paged(q, k, v, cos_sin, positions, slots, k_cache, v_cache, *, interleaved: bool = False,
                        want_k: bool = False):
    """Rotate queries and keys by their positions and append keys and values to a paged cache, in one launch.

    ``q [T,Hq,D]``, ``k`` and ``v [T,Hkv,D]`` fp16 or bf16, strided views (of one concatenated projection) included.
    ``cos_sin`` fp32 ``[positions, rotated]``: a row holds the cosines of a position's ``rotated / 2`` angles, then their
    sines; the first ``rotated`` values of a head turn, in pairs ``(i, i + rotated / 2)`` or, with ``interleaved``,
    ``(2i, 2i + 1)``.  Token ``t`` goes to offset ``slots[t] % page_size`` of page ``slots[t] // page_size`` of
    ``k_cache`` / ``v_cache [pages, Hkv, page_size, D]`` (views with other strides included), or nowhere where
    ``slots[t] < 0`` (padding); a slot may occur once per call (of two tokens with the same one, parts of either may be
    stored).  Views that share memory -- the two caches, a cache's entries, tokens within a cache -- raise ``ValueError``.
    ``positions`` and ``slots`` are int32 ``[T]``.  Inference only, as the attention operators: no gradients.

    Returns ``(q_rotated, k_rotated | None)``; the caches are updated in place.  Positions and slots out of range touch no
    memory and raise at the next :func:`check_device_errors`.
    """
    word = _index_word(_on_gpu(q, "q"))
    made = _lib.host().rotary_append(q, k, v, cos_sin, positions, slots, k_cache, v_cache, interleaved, want_k, word)
    if isinstance(made, int):
        _lib.check(made, "rotary_append_paged", q=tuple(q.shape), cache=tuple(k_cache.shape))
    return made


def paged_attention_decode(q, k_cache, v_cache, page_table, seq_lens, *, scale: float | None = None, out=None):
    """Attention of one new token per sequence over the pages its row of ``page_table`` names.

    ``q [B,Hq,D]`` fp16 or bf16, ``k_cache`` / ``v_cache [pages, Hkv, page_size, D]`` of the same type (``Hq`` a multiple of
    ``Hkv``), ``page_table`` int32 ``[B, pages of the longest]``, ``seq_lens`` int32 ``[B]``: tokens in the cache, the new
    one included; 0 gives a zero row.  What lies behind a sequence's end, in its last page and in its row of the table, is
    never read.  ``scale`` defaults to ``D ** -0.5``; ``out`` may be ``q``, where that is contiguous.  Softmax and sums run in
    fp32, the weights are rounded to the type before the product with the values.  Nothing depends on lengths known to the
    host: a captured call serves whatever lengths the tensor holds at replay.  Pages and lengths out of range raise at the next
    :func:`check_device_errors`; so may lengths that add up to half a billion tokens times ``Hkv`` (times sixteens of queries
    to a head of keys) within ``ceil(B / 256)`` neighbouring sequences, and then no row of the result is written.
    """
    word = _index_word(_on_gpu(q, "q"))
    y = _lib.host().paged_decode(q, k_cache, v_cache, page_table, seq_lens, scale, out, word)
    if isinstance(y, int):
        _lib.check(y, "paged_attention_decode", q=tuple(q.shape), cache=tuple(k_cache.shape))
    return y


def attention_prefill(q, k, v, cu_seqlens, *, scale: float | None = None, out=None):
    """Causal attention within packed sequences: rows ``cu_seqlens[b]`` to ``cu_seqlens[b + 1]`` are sequence ``b``.

    ``q [T,Hq,D]``, ``k`` and ``v [T,Hkv,D]`` fp16 or bf16, strided views included, ``Hq`` a multiple of ``Hkv``;
    ``cu_seqlens`` int32 ``[B + 1]``, ascending, at most ``T``.  Arithmetic as in :func:`paged_attention_decode`.  Returns ``out [T,Hq,D]``; rows that belong to no sequence
    are left as they are in ``out``, and unspecified without one.  ``scale`` defaults to ``D ** -0.5``; ``out`` may be ``q``,
    where that is contiguous.  Ends out of range or order leave all of ``out`` unspecified and raise at the next
    :func:`check_device_errors`.
    """
    device = _on_gpu(q, "q")
    y = _lib.host().attention_prefill(q, k, v, cu_seqlens, scale, out, _index_word(device), _error_word(device).data_ptr())
    if isinstance(y, int):
        _lib.check(y, "attention_prefill", q=tuple(q.shape), k=tuple(k.shape))
    return y
