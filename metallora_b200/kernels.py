"""Kernel-level API over the C ABI, taking and returning ``torch.Tensor``.

Mirrors the reference's kernel module (python/metal_lora/kernels.py): the same
entry-point names (``is_metal_available``, ``lora_forward_metal``,
``lora_backward_metal``, ``lora_adamw_step_metal``,
``persistent_gpu_state_init/step``), backed by sm_100a CUDA kernels instead of
Metal shaders.  Every call enqueues on the current torch CUDA stream and never
synchronises; workspaces come from torch's caching allocator.

Activations and weights are bf16 or fp16 (fp32 accumulation), or fp32, which
runs as split-precision bf16 tensor-core GEMMs (three partial products per
product of two fp32 values, ~2^-16 relative error each).
"""
from __future__ import annotations

import functools

import torch

from . import _lib
from .exceptions import ConfigurationError, DeviceError, ShapeError

_DT = {torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_F16, torch.float32: _lib.DTYPE_F32}


# the current stream's handle without building a Stream object (~3 us a call)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
_raw_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def _stream() -> int:
    if _raw_stream is not None:
        return _raw_stream(_raw_device())
    return torch.cuda.current_stream().cuda_stream


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def _need_cuda(*ts: torch.Tensor) -> None:
    for t in ts:
        if t is not None and not t.is_cuda:
            raise DeviceError("metallora_b200 kernels take CUDA tensors (no CPU fallback)")


def _need_current(*ts: torch.Tensor) -> None:
    """Launches go to the current device: tensors of another one are refused."""
    cur = torch.cuda.current_device()
    for t in ts:
        if t is not None and t.get_device() != cur:
            raise DeviceError(f"tensor on {t.device}, but cuda:{cur} is the current device")


def _need_here(first: torch.Tensor, *others: torch.Tensor | None) -> None:
    """``_need_cuda`` and ``_need_current`` of all of them, short where they hold."""
    d = first.get_device()
    for t in others:
        if t is not None and t.get_device() != d:
            d = -1
    if d < 0 or d != _raw_device():
        _need_cuda(first, *others)
        _need_current(first, *(t for t in others if t is not None))


def _dtype_code(t: torch.Tensor) -> int:
    try:
        return _DT[t.dtype]
    except KeyError:
        raise ShapeError(f"unsupported dtype {t.dtype}; use bfloat16, float16 or float32") from None


def _workspace(nbytes: int, device) -> torch.Tensor:
    return torch.empty(max(int(nbytes), 256), dtype=torch.uint8, device=device)


@functools.lru_cache(maxsize=256)
def _mx_ws_bytes(M: int, K: int, N: int, r: int, backward: bool, need_w: bool) -> int:
    """Workspace of a call over an MXFP4 base (a function of the sizes alone)."""
    lib = _lib.load()
    args = (M, K, N, r, _lib.QUANT_MXFP4, 32)
    if not backward:
        return lib.mlora_qlora_forward_workspace_bytes(*args)
    return (lib.mlora_qlora_backward_workspace_bytes(*args) if need_w
            else lib.mlora_qlora_lean_workspace_bytes(*args, 1))


@functools.lru_cache(maxsize=256)
def _bwd_ws_bytes(M: int, K: int, N: int, r: int, code: int) -> int:
    return _lib.load().mlora_lora_backward_workspace_bytes(M, K, N, r, code)


def is_metal_available() -> bool:
    """True when the CUDA extension loads and the current device is sm_100.

    Same name and meaning as the reference's ``kernels.is_metal_available()``
    (kernels.py:502): "can the custom kernels run here"."""
    try:
        lib = _lib.load()
    except DeviceError:
        return False
    if not torch.cuda.is_available():
        return False
    return bool(lib.mlora_device_supported(torch.cuda.current_device()))


def rank_tile(r: int) -> int:
    """Padded rank the tensor-core kernels use (power of two >= 16)."""
    R = 16
    while R < r:
        R *= 2
    return R


def _pad_rank(a: torch.Tensor, b: torch.Tensor, alpha: float):
    """Zero-pads A [r, K] / B [N, r] to a multiple-of-8 rank (16-byte rows) and
    rescales alpha so that alpha'/r' == alpha/r.  Zero rows/columns add nothing."""
    r = a.shape[0]
    r8 = (r + 7) // 8 * 8
    if r8 == r:
        return a, b, alpha, r
    a_p = torch.zeros((r8, a.shape[1]), dtype=a.dtype, device=a.device)
    a_p[:r] = a
    b_p = torch.zeros((b.shape[0], r8), dtype=b.dtype, device=b.device)
    b_p[:, :r] = b
    return a_p, b_p, alpha * r8 / r, r8


def _check_2d(name: str, t: torch.Tensor, shape: tuple, dtype: torch.dtype) -> None:
    if tuple(t.shape) != tuple(shape):
        raise ShapeError(f"{name} shape mismatch: expected {tuple(shape)}, got {tuple(t.shape)}")
    if t.dtype != dtype:
        raise ShapeError(f"{name} dtype mismatch: expected {dtype}, got {t.dtype}")


def lora_linear_fwd(x2d: torch.Tensor, w0: torch.Tensor, a: torch.Tensor, b: torch.Tensor,
                    alpha: float, save_xa: bool = False, ckpt_out=None):
    """y = x.W0^T + (alpha/r).(x.A^T).B^T for 2-D x [M, K].

    Returns (y, saved_xa); saved_xa is the [R, ceil8(M)] rank intermediate the
    backward can reuse (bf16/fp16 only), else None.  ``ckpt_out`` (a
    ``quant.empty_checkpoint`` of x) receives x's MXINT8 checkpoint."""
    _need_cuda(x2d, w0, a, b)
    dt = x2d.dtype
    code = _dtype_code(x2d)
    M, K = x2d.shape
    N = w0.shape[0]
    a, b, alpha, r = _pad_rank(a, b, alpha)
    _check_2d("W0", w0, (N, K), dt)
    _check_2d("A", a, (r, K), dt)
    _check_2d("B", b, (N, r), dt)
    x2d, w0, a, b = (t.contiguous() for t in (x2d, w0, a, b))
    y = x2d.new_empty((M, N))
    saved = None
    if save_xa and dt != torch.float32:
        saved = x2d.new_empty((rank_tile(r), (M + 7) // 8 * 8))
    if M == 0:  # no tokens: empty output, nothing to launch
        return y, saved
    lib = _lib.load()
    ws = _workspace(lib.mlora_lora_forward_workspace_bytes(M, K, N, r, code), x2d.device)
    head = (_ptr(x2d), _ptr(w0), _ptr(a), _ptr(b), _ptr(y), _ptr(saved))
    tail = (M, K, N, r, float(alpha), code, _ptr(ws), ws.numel(), _stream())
    if ckpt_out is not None:
        _check_ckpt_out(ckpt_out, x2d)
        st = lib.mlora_lora_forward_ckpt(*head, *_ckpt_args(ckpt_out), *tail)
    else:
        st = lib.mlora_lora_forward(*head, *tail)
    _lib.check(st, "mlora_lora_forward")
    return y, saved


def _as_ckpt(x, saved_xa, dy2d):
    """``x`` if it is an activation checkpoint the backward can take, else None."""
    if torch.is_tensor(x):
        return None
    x.check()
    _need_cuda(dy2d, x.codes)
    _need_current(dy2d, x.codes)
    if x.dtype not in (torch.bfloat16, torch.float16):
        raise ShapeError("a checkpointed backward takes bf16/fp16 activations")
    if saved_xa is None:
        raise ShapeError("a checkpointed backward needs the forward's saved_xa")
    return x


def _ckpt_args(ckpt):
    return _ptr(ckpt.codes), ckpt.codes.stride(0), _ptr(ckpt.scales)


def _check_ckpt_out(ckpt, x2d) -> None:
    ckpt.check()
    if (ckpt.rows, ckpt.shape[-1], ckpt.dtype, ckpt.device) != (*x2d.shape, x2d.dtype, x2d.device):
        raise ShapeError("the checkpoint to fill does not match x")
    _need_current(x2d)


def _check_saved(saved_xa, r: int, M: int, dtype: torch.dtype) -> None:
    _check_2d("saved_xa", saved_xa, (rank_tile(r), (M + 7) // 8 * 8), dtype)
    _need_cuda(saved_xa)
    if not saved_xa.is_contiguous():
        raise ShapeError("saved_xa must be contiguous")


def _check_grad_out(da_out, db_out, r: int, r_orig: int, K: int, N: int) -> None:
    if r != r_orig:
        raise ShapeError("gradient accumulation buffers need a rank that is a multiple of 8")
    for name, t, shp in (("da_out", da_out, (r, K)), ("db_out", db_out, (N, r))):
        if t is None or t.dtype != torch.float32 or tuple(t.shape) != shp or \
                not t.is_contiguous():
            raise ShapeError(f"{name} must be a contiguous fp32 tensor of shape {shp}")
    _need_cuda(da_out, db_out)


def lora_linear_bwd(dy2d: torch.Tensor, x2d: torch.Tensor, w0: torch.Tensor | None,
                    a: torch.Tensor, b: torch.Tensor, alpha: float,
                    saved_xa: torch.Tensor | None = None, clip_value: float = 0.0,
                    need_dx: bool = True, da_out: torch.Tensor | None = None,
                    db_out: torch.Tensor | None = None, accumulate: bool = True,
                    grad_dtype: torch.dtype | None = None):
    """(dx, dA, dB) of the LoRA linear for 2-D dy [M, N], x [M, K].

    dA/dB are fp32 (master-gradient precision), or x's 16-bit dtype when
    ``grad_dtype`` names it (written by the kernel, no cast launch); clip_value
    > 0 clips them elementwise after the full reduction (ops.py:155).  With ``da_out`` and
    ``db_out`` (contiguous fp32 [r, K] / [N, r], rank a multiple of 8) the
    gradients are ADDED into those buffers (written over them when
    ``accumulate`` is False) and returned.  ``x2d`` may be an MXINT8
    ``quant.ActivationCheckpoint`` of x: dA is then taken from its values, and
    ``saved_xa`` is required."""
    ckpt = _as_ckpt(x2d, saved_xa, dy2d)
    _need_cuda(dy2d, a, b) if ckpt is not None else _need_cuda(dy2d, x2d, a, b)
    dt = x2d.dtype
    code = _dtype_code(x2d)
    M, K = x2d.shape if ckpt is None else (ckpt.rows, ckpt.shape[-1])
    N = dy2d.shape[1]
    r_orig = a.shape[0]
    a_p, b_p, alpha_p, r = _pad_rank(a, b, alpha)
    if dt == torch.float32:
        saved_xa = None
    _check_2d("grad_output", dy2d, (M, N), dt)
    _check_2d("A", a_p, (r, K), dt)
    _check_2d("B", b_p, (N, r), dt)
    if saved_xa is not None:
        _check_saved(saved_xa, r, M, dt)
    if need_dx:
        if w0 is None:
            raise ShapeError("dx needs W0")
        _check_2d("W0", w0, (N, K), dt)
        w0 = w0.contiguous()
    dy2d, a_p, b_p = dy2d.contiguous(), a_p.contiguous(), b_p.contiguous()
    if ckpt is None:
        x2d = x2d.contiguous()
    lib = _lib.load()
    dx = dy2d.new_empty((M, K)) if need_dx else None
    flags = 0
    into = da_out is not None or db_out is not None
    if into:
        _check_grad_out(da_out, db_out, r, r_orig, K, N)
        da, db = da_out, db_out
        flags = _lib.BWD_ACCUMULATE if accumulate else 0
    else:
        if grad_dtype is not None and grad_dtype == dt and dt != torch.float32:
            flags = _lib.BWD_GRADS_16BIT
            da, db = dy2d.new_empty((r, K)), dy2d.new_empty((N, r))
        else:
            da = dy2d.new_empty((r, K), dtype=torch.float32)
            db = dy2d.new_empty((N, r), dtype=torch.float32)
    if M == 0:  # no tokens: the sums over tokens are zero; nothing to launch
        if not (into and accumulate):
            da.zero_()
            db.zero_()
        if into:
            return dx, da, db
        return dx, da[:r_orig].contiguous(), db[:, :r_orig].contiguous()
    ws = dy2d.new_empty(_bwd_ws_bytes(M, K, N, r, code), dtype=torch.uint8)
    tail = (_ptr(w0) if need_dx else None, _ptr(a_p), _ptr(b_p), _ptr(saved_xa), _ptr(dx), _ptr(da),
            _ptr(db), M, K, N, r, float(alpha_p), float(clip_value), code, flags, _ptr(ws),
            ws.numel(), _stream())
    if ckpt is not None:
        st = lib.mlora_lora_backward_ckpt(_ptr(dy2d), *_ckpt_args(ckpt), *tail)
    else:
        st = lib.mlora_lora_backward_ex(_ptr(dy2d), _ptr(x2d), *tail)
    _lib.check(st, "mlora_lora_backward")
    if into:
        return dx, da, db
    if r != r_orig:
        da, db = da[:r_orig].contiguous(), db[:, :r_orig].contiguous()
    return dx, da, db


def lora_linear_bwd_split(dy2d: torch.Tensor, x2d: torch.Tensor, w0: torch.Tensor,
                          a: torch.Tensor, b: torch.Tensor, alpha: float,
                          saved_xa: torch.Tensor | None, da_out: torch.Tensor,
                          db_out: torch.Tensor, accumulate: bool = True):
    """The 16-bit backward in two launches (MLORA_BWD_DEFER_DX, then
    MLORA_BWD_DX_ONLY): enqueues everything but the dx GEMM -- dA/dB land in
    ``da_out``/``db_out`` (fp32, added or written as ``accumulate`` says) --
    and returns ``finish``, which enqueues the dx GEMM and returns dx.  Work
    that needs only dA/dB (a gradient exchange on another stream) can be
    started between the two and overlaps the GEMM.  ``x2d`` may be an activation
    checkpoint, as for ``lora_linear_bwd``."""
    ckpt = _as_ckpt(x2d, saved_xa, dy2d)
    _need_cuda(dy2d, a, b) if ckpt is not None else _need_cuda(dy2d, x2d, a, b)
    dt = x2d.dtype
    if dt == torch.float32:
        raise ShapeError("the split backward takes bf16/fp16 tensors")
    code = _dtype_code(x2d)
    M, K = x2d.shape if ckpt is None else (ckpt.rows, ckpt.shape[-1])
    N = dy2d.shape[1]
    r = a.shape[0]
    if r % 8:
        raise ShapeError("gradient buffers need a rank that is a multiple of 8")
    _check_2d("grad_output", dy2d, (M, N), dt)
    _check_2d("W0", w0, (N, K), dt)
    _check_2d("A", a, (r, K), dt)
    _check_2d("B", b, (N, r), dt)
    _check_grad_out(da_out, db_out, r, r, K, N)
    dy2d, w0, a, b = (t.contiguous() for t in (dy2d, w0, a, b))
    if ckpt is None:
        x2d = x2d.contiguous()
    if saved_xa is not None:
        _check_saved(saved_xa, r, M, dt)
    lib = _lib.load()
    dx = torch.empty((M, K), dtype=dt, device=x2d.device)
    ws = _workspace(lib.mlora_lora_backward_workspace_bytes(M, K, N, r, code), x2d.device)
    flags = _lib.BWD_ACCUMULATE if accumulate else 0
    if M == 0:  # no tokens: zero gradients (unless added to), empty dx
        if not accumulate:
            da_out.zero_()
            db_out.zero_()
        return lambda: dx

    def call(phase):
        tail = (_ptr(w0), _ptr(a), _ptr(b), _ptr(saved_xa), _ptr(dx), _ptr(da_out), _ptr(db_out),
                M, K, N, r, float(alpha), 0.0, code, flags | phase, _ptr(ws), ws.numel(), _stream())
        if ckpt is not None:
            st = lib.mlora_lora_backward_ckpt(_ptr(dy2d), *_ckpt_args(ckpt), *tail)
        else:
            st = lib.mlora_lora_backward_ex(_ptr(dy2d), _ptr(x2d), *tail)
        _lib.check(st, "mlora_lora_backward_ex")

    call(_lib.BWD_DEFER_DX)

    def finish() -> torch.Tensor:
        call(_lib.BWD_DX_ONLY)
        return dx
    return finish


def linear(x2d: torch.Tensor, w: torch.Tensor) -> torch.Tensor:
    """y = x.W^T (merged-weight forward, ops.py:106-114)."""
    _need_cuda(x2d, w)
    code = _dtype_code(x2d)
    M, K = x2d.shape
    N = w.shape[0]
    _check_2d("W", w, (N, K), x2d.dtype)
    x2d, w = x2d.contiguous(), w.contiguous()
    y = torch.empty((M, N), dtype=x2d.dtype, device=x2d.device)
    if M == 0:
        return y
    lib = _lib.load()
    ws = _workspace(lib.mlora_linear_workspace_bytes(M, K, N, code), x2d.device)
    st = lib.mlora_linear(_ptr(x2d), _ptr(w), _ptr(y), M, K, N, code, _ptr(ws), ws.numel(),
                          _stream())
    _lib.check(st, "mlora_linear")
    return y


def merge(w0: torch.Tensor, a: torch.Tensor, b: torch.Tensor, alpha: float,
          out: torch.Tensor | None = None) -> torch.Tensor:
    """W0 + (alpha/r).B.A (ops.py:162-172); ``out`` may be ``w0`` (in place)."""
    _need_cuda(w0, a, b)
    code = _dtype_code(w0)
    N, K = w0.shape
    a_p, b_p, alpha_p, r = _pad_rank(a, b, alpha)
    _check_2d("A", a_p, (r, K), w0.dtype)
    _check_2d("B", b_p, (N, r), w0.dtype)
    w0, a_p, b_p = w0.contiguous(), a_p.contiguous(), b_p.contiguous()
    lib = _lib.load()
    if out is None:
        out = torch.empty_like(w0)
    ws = _workspace(lib.mlora_merge_workspace_bytes(N, K, r, code), w0.device)
    st = lib.mlora_merge(_ptr(w0), _ptr(a_p), _ptr(b_p), _ptr(out), N, K, r, float(alpha_p), code,
                         _ptr(ws), ws.numel(), _stream())
    _lib.check(st, "mlora_merge")
    return out


def lora_forward_metal(x, w0, a, b, alpha: float = 16.0, batch_size=None, seq_len=None,
                       use_simd=None):
    """Fused LoRA forward (reference: kernels.py:507-566).  x is [B, S, K] or
    [S, K]; batch_size/seq_len/use_simd are accepted for signature parity."""
    shp = x.shape
    y, _ = lora_linear_fwd(x.reshape(-1, shp[-1]), w0, a, b, alpha)
    return y.reshape(*shp[:-1], w0.shape[0])


def lora_backward_metal(grad_output, x, a, b, alpha: float = 16.0, clip_value: float = 1.0):
    """(grad_A, grad_B) of the LoRA branch, clipped to +-clip_value (reference:
    kernels.py:569-612 / ops.py:143-155), returned in A's/B's dtype."""
    g = grad_output.reshape(-1, grad_output.shape[-1])
    xx = x.reshape(-1, x.shape[-1])
    _, da, db = lora_linear_bwd(g, xx, None, a, b, alpha, None, clip_value, need_dx=False)
    return da.to(a.dtype), db.to(b.dtype)


# ------------------------------------------------------------------ optimizer --

def persistent_gpu_state_init(beta1: float = 0.9, beta2: float = 0.999, device=None):
    """Device Adam state [step, beta1^step, beta2^step] (kernels.py:471-481).

    Starts at step 0 ([0, 1, 1]); ``persistent_gpu_state_step`` advances it
    before each update, so the first update uses step 1 and beta^1 -- the
    formula tests/test_parity.py:57-64 pins.  (The reference initialises to
    [1, b1, b2] and also steps before the first update, so its first update
    uses beta^2.)"""
    dev = device if device is not None else torch.device("cuda", torch.cuda.current_device())
    return torch.tensor([0.0, 1.0, 1.0], dtype=torch.float32, device=dev)


def persistent_gpu_state_step(gpu_state: torch.Tensor, beta1: float = 0.9, beta2: float = 0.999):
    """state := [t+1, b1^(t+1), b2^(t+1)] on the device (kernels.py:484-499)."""
    _need_cuda(gpu_state)
    _lib.check(_lib.load().mlora_adam_state_step(_ptr(gpu_state), beta1, beta2, _stream()),
               "mlora_adam_state_step")


def lora_adamw_step_metal(param, grad, m, v, gpu_state, lr: float, beta1: float, beta2: float,
                          eps: float, wd: float, grad_scale: torch.Tensor | None = None):
    """In-place AdamW step (kernels.py:615-643): updates param, m, v and zeroes
    grad.  param bf16/fp16/fp32; grad, m, v fp32 and contiguous."""
    _need_cuda(param, grad, m, v, gpu_state)
    for name, t in (("grad", grad), ("m", m), ("v", v)):
        if t.dtype != torch.float32 or t.numel() != param.numel() or not t.is_contiguous():
            raise ShapeError(f"{name} must be contiguous fp32 with param's size")
    if not param.is_contiguous():
        raise ShapeError("param must be contiguous")
    st = _lib.load().mlora_adamw_step(_ptr(param), _ptr(grad), _ptr(m), _ptr(v), _ptr(gpu_state),
                                      param.numel(), lr, beta1, beta2, eps, wd,
                                      _dtype_code(param), _ptr(grad_scale), _stream())
    _lib.check(st, "mlora_adamw_step")


def sgd_step(param, grad, lr: float, grad_scale: torch.Tensor | None = None):
    """In-place p -= lr * g (zeroes grad)."""
    _need_cuda(param, grad)
    st = _lib.load().mlora_sgd_step(_ptr(param), _ptr(grad), param.numel(), lr, _dtype_code(param),
                                    _ptr(grad_scale), _stream())
    _lib.check(st, "mlora_sgd_step")


def grad_norm_clip(grad: torch.Tensor, max_norm: float, out: torch.Tensor | None = None):
    """Device [clip scale, norm] of a flat fp32 gradient (trainer.py:237-240)."""
    _need_cuda(grad)
    if grad.dtype != torch.float32 or not grad.is_contiguous():
        raise ShapeError("grad must be contiguous fp32")
    lib = _lib.load()
    if out is None:
        out = torch.empty(2, dtype=torch.float32, device=grad.device)
    ws = _workspace(lib.mlora_grad_norm_workspace_bytes(), grad.device)
    st = lib.mlora_grad_norm_clip(_ptr(grad), grad.numel(), float(max_norm), _ptr(out), _ptr(ws),
                                  ws.numel(), _stream())
    _lib.check(st, "mlora_grad_norm_clip")
    return out


# --------------------------------------------------------- quantised bases --

def _qlora_ws_bytes(lib, qw, M, K, N, r, backward, need_w=True):
    """Staged workspace (a bf16 copy of deq(W), fastest) unless the weight asks
    for the lean fused-dequant kernel, or the call does not read the weight."""
    if qw.scheme == "mxfp4":
        return _mx_ws_bytes(M, K, N, r, backward, need_w)
    if getattr(qw, "lean", False) or not need_w:
        return lib.mlora_qlora_lean_workspace_bytes(M, K, N, r, qw.code, qw.group, int(backward))
    fn = (lib.mlora_qlora_backward_workspace_bytes if backward
          else lib.mlora_qlora_forward_workspace_bytes)
    return fn(M, K, N, r, qw.code, qw.group)


def _qlora_dtype(x2d, qw) -> torch.dtype:
    """The activations' dtype, checked against what the base's scheme takes."""
    if getattr(qw, "scheme", None) == "mxfp4":
        if x2d.dtype not in (torch.bfloat16, torch.float16):
            raise ShapeError("an MXFP4 base takes bf16 or fp16 activations")
        _need_current(x2d if torch.is_tensor(x2d) else x2d.codes, qw.codes)
    elif x2d.dtype != torch.bfloat16:
        raise ShapeError("quantised-base LoRA takes bf16 activations")
    return x2d.dtype


def qlora_linear_fwd(x2d: torch.Tensor, qw, a: torch.Tensor, b: torch.Tensor, alpha: float,
                     save_xa: bool = False, ckpt_out=None):
    """y = x.deq(W)^T + (alpha/r).(x.A^T).B^T for a quantised base ``qw``
    (metallora_b200.quant.QuantizedWeight); x, A, B bf16.  ``qw.lean`` selects
    the fused kernel that dequantises in its main loop (no dense copy of W).
    An MXFP4 base takes bf16 or fp16 and multiplies x rounded to MXFP4.
    ``ckpt_out`` as for ``lora_linear_fwd``."""
    _need_cuda(x2d, a, b)
    dt = _qlora_dtype(x2d, qw)
    M, K = x2d.shape
    N = qw.shape[0]
    if qw.shape[1] != K:
        raise ShapeError(f"x has {K} features, the quantised weight {qw.shape[1]}")
    a, b, alpha, r = _pad_rank(a, b, alpha)
    _check_2d("A", a, (r, K), dt)
    _check_2d("B", b, (N, r), dt)
    x2d, a, b = x2d.contiguous(), a.contiguous(), b.contiguous()
    y = x2d.new_empty((M, N))
    saved = x2d.new_empty((rank_tile(r), (M + 7) // 8 * 8)) if save_xa else None
    if M == 0:  # no tokens: empty output, nothing to launch
        return y, saved
    lib = _lib.load()
    ws = x2d.new_empty(_qlora_ws_bytes(lib, qw, M, K, N, r, backward=False), dtype=torch.uint8)
    zeros = qw.zeros
    head = (x2d.data_ptr(), qw.code, qw.codes.data_ptr(), qw.scales.data_ptr(),
            None if zeros is None else zeros.data_ptr(), qw.prepared_scales().data_ptr(), qw.group,
            a.data_ptr(), b.data_ptr(), y.data_ptr(), None if saved is None else saved.data_ptr())
    tail = (M, K, N, r, float(alpha), _DT[dt], ws.data_ptr(), ws.numel(), _stream())
    if ckpt_out is not None:
        _check_ckpt_out(ckpt_out, x2d)
        st = lib.mlora_qlora_forward_ckpt(*head, *_ckpt_args(ckpt_out), *tail)
    else:
        st = lib.mlora_qlora_forward_ex(*head, *tail)
    _lib.check(st, "mlora_qlora_forward_ex")
    return y, saved


def qlora_linear_bwd(dy2d: torch.Tensor, x2d: torch.Tensor, qw, a: torch.Tensor, b: torch.Tensor,
                     alpha: float, saved_xa: torch.Tensor | None = None, clip_value: float = 0.0,
                     need_dx: bool = True, da_out: torch.Tensor | None = None,
                     db_out: torch.Tensor | None = None, accumulate: bool = True,
                     grad_dtype: torch.dtype | None = None):
    """(dx, dA, dB) through a frozen quantised base (staged or lean as the forward);
    ``da_out``/``db_out``/``accumulate``/``grad_dtype`` and an activation
    checkpoint in the place of ``x2d`` as in ``lora_linear_bwd``."""
    ckpt = _as_ckpt(x2d, saved_xa, dy2d)
    _need_cuda(dy2d, a, b) if ckpt is not None else _need_cuda(dy2d, x2d, a, b)
    dt = _qlora_dtype(x2d, qw)
    M, K = x2d.shape if ckpt is None else (ckpt.rows, ckpt.shape[-1])
    N = dy2d.shape[1]
    if tuple(qw.shape) != (N, K):
        raise ShapeError(f"the quantised weight is {tuple(qw.shape)}, grad_output and x are of "
                         f"{(N, K)}")
    r_orig = a.shape[0]
    a_p, b_p, alpha_p, r = _pad_rank(a, b, alpha)
    _check_2d("grad_output", dy2d, (M, N), dt)
    _check_2d("A", a_p, (r, K), dt)
    _check_2d("B", b_p, (N, r), dt)
    dy2d, a_p, b_p = dy2d.contiguous(), a_p.contiguous(), b_p.contiguous()
    if ckpt is None:
        x2d = x2d.contiguous()
    if saved_xa is not None:
        _check_saved(saved_xa, r, M, dt)
    lib = _lib.load()
    dx = dy2d.new_empty((M, K)) if need_dx else None
    flags = 0
    into = da_out is not None or db_out is not None
    if into:
        _check_grad_out(da_out, db_out, r, r_orig, K, N)
        da, db = da_out, db_out
        flags = _lib.BWD_ACCUMULATE if accumulate else 0
    else:
        if grad_dtype is not None and grad_dtype == dt:
            flags = _lib.BWD_GRADS_16BIT
            da, db = dy2d.new_empty((r, K)), dy2d.new_empty((N, r))
        else:
            da = dy2d.new_empty((r, K), dtype=torch.float32)
            db = dy2d.new_empty((N, r), dtype=torch.float32)
    if M == 0:  # no tokens: the sums over tokens are zero; nothing to launch
        if not (into and accumulate):
            da.zero_()
            db.zero_()
        if into:
            return dx, da, db
        return dx, da[:r_orig].contiguous(), db[:, :r_orig].contiguous()
    ws = dy2d.new_empty(_qlora_ws_bytes(lib, qw, M, K, N, r, backward=True, need_w=need_dx),
                        dtype=torch.uint8)
    tail = (qw.code, qw.codes.data_ptr(), qw.scales.data_ptr(), _ptr(qw.zeros),
            _ptr(qw.prepared_scales()) if need_dx and qw.scheme != "mxfp4" else None, qw.group,
            a_p.data_ptr(), b_p.data_ptr(), _ptr(saved_xa), _ptr(dx), da.data_ptr(),
            db.data_ptr(), M, K, N, r, float(alpha_p), float(clip_value), _DT[dt], flags,
            ws.data_ptr(), ws.numel(), _stream())
    if ckpt is not None:
        st = lib.mlora_qlora_backward_ckpt(_ptr(dy2d), *_ckpt_args(ckpt), *tail)
    else:
        st = lib.mlora_qlora_backward_ex(_ptr(dy2d), _ptr(x2d), *tail)
    _lib.check(st, "mlora_qlora_backward_ex")
    if into:
        return dx, da, db
    if r != r_orig:
        da, db = da[:r_orig].contiguous(), db[:, :r_orig].contiguous()
    return dx, da, db


# ------------------------------------------------------ stacked adapters --

MAX_STACKED_RANK = 256  # n_adapters * rank per launch


def multi_lora_fwd(x2d: torch.Tensor, w0: torch.Tensor | None, a_stack: torch.Tensor,
                   b_stack: torch.Tensor, ids: torch.Tensor, r: int, alpha: float) -> torch.Tensor:
    """y = (x.w0^T if w0 is given) + (alpha/r) (x.A_g^T).B_g^T with g = ids[m] per
    token, over n adapters stacked as a_stack [n*r, K] and b_stack [N, n*r]
    (one launch of the rank kernel for all of them, then the tcgen05 GEMM);
    ids is an int32 CUDA tensor [M]; an id outside [0, n) adds no LoRA term."""
    _need_cuda(x2d, a_stack, b_stack, ids, w0)
    M, K = x2d.shape
    nr, K2 = a_stack.shape
    N = b_stack.shape[0]
    if K2 != K or b_stack.shape[1] != nr or nr % r:
        raise ShapeError("a_stack [n*r, K] and b_stack [N, n*r] do not match x / r")
    if w0 is not None:
        _check_2d("W0", w0, (N, K), x2d.dtype)
    if ids.dtype != torch.int32 or ids.numel() != M:
        raise ShapeError("ids must be an int32 tensor with one entry per token")
    n = nr // r
    x2d, a_stack, b_stack = x2d.contiguous(), a_stack.contiguous(), b_stack.contiguous()
    y = torch.empty((M, N), dtype=x2d.dtype, device=x2d.device)
    if M == 0:
        return y
    lib = _lib.load()
    code = _dtype_code(x2d)
    ws = _workspace(lib.mlora_multi_lora_forward_workspace_bytes(M, K, N, r, n, code), x2d.device)
    st = lib.mlora_multi_lora_forward(_ptr(x2d), _ptr(w0), _ptr(a_stack), _ptr(b_stack),
                                      _ptr(ids.contiguous()), _ptr(y), M, K, N, r, n, float(alpha),
                                      code, _ptr(ws), ws.numel(), _stream())
    _lib.check(st, "mlora_multi_lora_forward")
    return y


# ------------------------------------------------------------ embedding --

def _as_idx(indices: torch.Tensor) -> torch.Tensor:
    return indices.reshape(-1).to(torch.int32).contiguous()


def lora_embedding_fwd(indices: torch.Tensor, table: torch.Tensor, a: torch.Tensor,
                       b: torch.Tensor, alpha: float) -> torch.Tensor:
    """table[idx] + (alpha/r) b[idx].a for every index (LoRAEmbedding.__call__,
    layers.py:220-225); returns [*indices.shape, D]."""
    _need_cuda(indices, table, a, b)
    V, D = table.shape
    r = a.shape[0]
    _check_2d("A", a, (r, D), table.dtype)
    _check_2d("B", b, (V, r), table.dtype)
    idx = _as_idx(indices)
    T = idx.numel()
    code = _dtype_code(table)
    out = torch.empty((T, D), dtype=table.dtype, device=table.device)
    if T == 0:
        return out.reshape(*indices.shape, D)
    lib = _lib.load()
    ws = _workspace(lib.mlora_lora_embedding_workspace_bytes(T, D, r, code, 0), table.device)
    st = lib.mlora_lora_embedding_forward(_ptr(idx), _ptr(table.contiguous()), _ptr(a.contiguous()),
                                          _ptr(b.contiguous()), _ptr(out), T, V, D, r, float(alpha),
                                          code, _ptr(ws), ws.numel(), _stream())
    _lib.check(st, "mlora_lora_embedding_forward")
    return out.reshape(*indices.shape, D)


def lora_embedding_bwd(dy: torch.Tensor, indices: torch.Tensor, a: torch.Tensor, b: torch.Tensor,
                       alpha: float, da_out: torch.Tensor | None = None,
                       db_out: torch.Tensor | None = None):
    """fp32 (dA [r, D], dB [V, r]) of the LoRA embedding; dB rows are summed over
    each index's tokens in token order (deterministic).  With da_out/db_out the
    gradients are added into them."""
    _need_cuda(dy, indices, a, b)
    V, r = b.shape
    D = a.shape[1]
    idx = _as_idx(indices)
    T = idx.numel()
    dy2 = dy.reshape(T, D).contiguous()
    sorted_idx, order = torch.sort(idx, stable=True)
    order = order.to(torch.int32)
    lib = _lib.load()
    code = _dtype_code(dy2)
    flags = 0
    if da_out is not None and db_out is not None:
        da, db, flags = da_out, db_out, _lib.BWD_ACCUMULATE
    else:
        da = torch.empty((r, D), dtype=torch.float32, device=dy.device)
        db = torch.empty((V, r), dtype=torch.float32, device=dy.device)
    if T == 0:  # no tokens: zero gradients (or nothing added); nothing to launch
        if not flags:
            da.zero_()
            db.zero_()
        return da, db
    ws = _workspace(lib.mlora_lora_embedding_workspace_bytes(T, D, r, code, 1), dy.device)
    st = lib.mlora_lora_embedding_backward(_ptr(dy2), _ptr(idx), _ptr(sorted_idx), _ptr(order),
                                           _ptr(a.contiguous()), _ptr(b.contiguous()), _ptr(da),
                                           _ptr(db), T, V, D, r, float(alpha), code, flags,
                                           _ptr(ws), ws.numel(), _stream())
    _lib.check(st, "mlora_lora_embedding_backward")
    return da, db


# ------------------------------------------------------- KV-cache update --

def lora_kv_cache_update(x2d: torch.Tensor, wk: torch.Tensor, wv: torch.Tensor, ak: torch.Tensor,
                         bk: torch.Tensor, av: torch.Tensor, bv: torch.Tensor,
                         k_cache: torch.Tensor, v_cache: torch.Tensor, cur_pos: int,
                         alpha: float) -> None:
    """Projects one new token per sequence through the K and V LoRA linears and
    writes the rows straight into k_cache/v_cache [batch, max_seq, ...] at
    position cur_pos (lora_kv_cache_update, kernels/lora_kernels.metal:514-586)."""
    _need_cuda(x2d, wk, wv, ak, bk, av, bv, k_cache, v_cache)
    batch, D_in = x2d.shape
    D_kv = wk.shape[0]
    max_seq = k_cache.shape[1]
    if k_cache.shape[0] != batch or k_cache[0, 0].numel() != D_kv or v_cache.shape != k_cache.shape:
        raise ShapeError("caches must be [batch, max_seq, D_kv] (trailing dims may be heads, dim)")
    if not (k_cache.is_contiguous() and v_cache.is_contiguous()):
        raise ShapeError("caches must be contiguous")
    r_orig = ak.shape[0]
    ak, bk, alpha_k, r = _pad_rank(ak, bk, alpha)
    av, bv, _, _ = _pad_rank(av, bv, alpha)
    for name, t, shape in (("W_K", wk, (D_kv, D_in)), ("W_V", wv, (D_kv, D_in)),
                           ("A_K", ak, (r, D_in)), ("A_V", av, (r, D_in)),
                           ("B_K", bk, (D_kv, r)), ("B_V", bv, (D_kv, r))):
        _check_2d(name, t, shape, x2d.dtype)
    del r_orig
    if batch == 0:  # no sequences: nothing to write
        return
    lib = _lib.load()
    code = _dtype_code(x2d)
    ws = _workspace(lib.mlora_lora_kv_cache_workspace_bytes(batch, D_in, D_kv, r, code), x2d.device)
    st = lib.mlora_lora_kv_cache_update(
        _ptr(x2d.contiguous()), _ptr(wk.contiguous()), _ptr(wv.contiguous()), _ptr(ak.contiguous()),
        _ptr(bk.contiguous()), _ptr(av.contiguous()), _ptr(bv.contiguous()), _ptr(k_cache),
        _ptr(v_cache), batch, int(cur_pos), max_seq, D_in, D_kv, r, float(alpha_k), code, _ptr(ws),
        ws.numel(), _stream())
    _lib.check(st, "mlora_lora_kv_cache_update")


# --------------------------------------------------- linear cross entropy --

@functools.lru_cache(maxsize=256)
def _head_bytes(M: int, K: int, V: int, r: int, code: int, grads: int) -> tuple[int, int]:
    """(state, workspace) bytes of a linear cross entropy (a function of the sizes alone)."""
    lib = _lib.load()
    args = (M, K, V, r, code, grads)
    return (lib.mlora_linear_cross_entropy_state_bytes(*args),
            lib.mlora_linear_cross_entropy_workspace_bytes(*args))


def _head_dtype(x2d: torch.Tensor) -> int:
    if x2d.dtype not in (torch.bfloat16, torch.float16):
        raise ShapeError("the linear cross entropy takes bf16 or fp16 hidden states")
    return _DT[x2d.dtype]


def linear_cross_entropy_fwd(x2d: torch.Tensor, w: torch.Tensor, labels: torch.Tensor,
                             a: torch.Tensor | None = None, b: torch.Tensor | None = None,
                             alpha: float = 16.0, ignore_index: int = -100,
                             reduction: str = "mean", grads: int = 0):
    """Softmax cross entropy of the head ``x.W^T (+ (alpha/r)(x.A^T).B^T)`` for 2-D
    x [M, K], W [V, K] and labels [M].

    Returns (loss, state): loss fp32, a scalar or ("none") one per token; state
    holds the gradients that ``grads`` (``_lib.HEAD_GRAD_*``) names for a unit
    upstream gradient, for ``linear_cross_entropy_bwd``."""
    _need_here(x2d, w, labels, a, b)
    code = _head_dtype(x2d)
    M, K = x2d.shape
    V = w.shape[0]
    _check_2d("weight", w, (V, K), x2d.dtype)
    if labels.shape != (M,):
        raise ShapeError(f"labels shape mismatch: expected {(M,)}, got {tuple(labels.shape)}")
    if labels.dtype != torch.int64:
        if labels.dtype != torch.int32:
            raise ShapeError(f"labels must be int64 or int32, got {labels.dtype}")
        labels = labels.to(torch.int64)
    r = 0
    if a is not None:
        a, b, alpha, r = _pad_rank(a, b, alpha)
        _check_2d("A", a, (r, K), x2d.dtype)
        _check_2d("B", b, (V, r), x2d.dtype)
        a, b = a.contiguous(), b.contiguous()
    x2d, w, labels = x2d.contiguous(), w.contiguous(), labels.contiguous()
    rows = reduction == "none"
    loss = x2d.new_empty((M,) if rows else (), dtype=torch.float32)
    if M == 0:  # no tokens: nothing to launch (a mean over none is NaN, as 0 / 0 is)
        return loss.fill_(float("nan") if reduction == "mean" else 0.0), loss.new_empty(0)
    lib = _lib.load()
    state_bytes, ws_bytes = _head_bytes(M, K, V, r, code, grads)
    if state_bytes == 0:  # the sizes are refused: the call says why
        _lib.check(lib.mlora_linear_cross_entropy(*(None,) * 8, 0, M, K, V, r, float(alpha), 0, 0,
                                                  code, grads, None, 0, None),
                   "mlora_linear_cross_entropy")
    state = x2d.new_empty(state_bytes, dtype=torch.uint8)
    ws = x2d.new_empty(ws_bytes, dtype=torch.uint8)
    out = loss.data_ptr()
    st = lib.mlora_linear_cross_entropy(
        x2d.data_ptr(), w.data_ptr(), _ptr(a), _ptr(b), labels.data_ptr(), None if rows else out,
        out if rows else None, state.data_ptr(), state_bytes, M, K, V, r, float(alpha),
        int(ignore_index), reduction == "mean", code, grads, ws.data_ptr(), ws_bytes, _stream())
    _lib.check(st, "mlora_linear_cross_entropy")
    return loss, state


def linear_cross_entropy_bwd(grad: torch.Tensor, state: torch.Tensor, w: torch.Tensor, M: int,
                             r: int, reduction: str, grads: int,
                             da_out: torch.Tensor | None = None,
                             db_out: torch.Tensor | None = None, accumulate: bool = True,
                             ab_dtype: torch.dtype | None = None):
    """(dx, dA, dB, dW), those that ``grads`` names, from the state that
    ``linear_cross_entropy_fwd`` filled with the same ``grads``, and the loss's
    upstream gradient (fp32; one per token after "none").  r is A's rank.  With
    ``da_out``/``db_out`` (contiguous fp32, rank a multiple of 8) dA and dB are added
    into them, or written over them without ``accumulate``."""
    _need_here(grad, state, w)
    code = _head_dtype(w)
    V, K = w.shape
    r8 = (r + 7) // 8 * 8
    dx = w.new_empty((M, K)) if grads & _lib.HEAD_GRAD_X else None
    dw = torch.empty((V, K), dtype=w.dtype, device=w.device) if grads & _lib.HEAD_GRAD_W else None
    da = db = None
    into = da_out is not None or db_out is not None
    if grads & _lib.HEAD_GRAD_AB:
        if into:
            _check_grad_out(da_out, db_out, r8, r, K, V)
            da, db = da_out, db_out
        else:
            da = w.new_empty((r8, K), dtype=ab_dtype or w.dtype)
            db = w.new_empty((V, r8), dtype=ab_dtype or w.dtype)
    if M == 0:  # no tokens: zero gradients (or nothing added)
        for t in (dw, *(() if into and accumulate else (da, db))):
            if t is not None:
                t.zero_()
    else:
        w = w.contiguous()
        rows = reduction == "none"
        if grad.dtype != torch.float32:
            grad = grad.to(torch.float32)
        grad = grad.contiguous()
        if rows and tuple(grad.shape) != (M,):
            raise ShapeError(f"expected {M} upstream gradients, got {tuple(grad.shape)}")
        st = _lib.load().mlora_linear_cross_entropy_backward(
            state.data_ptr(), state.numel(), grad.data_ptr(), rows, reduction == "mean", w.data_ptr(),
            _ptr(dx), _ptr(da), _ptr(db), code if da is None else _dtype_code(da),
            int(into and accumulate), _ptr(dw), M, K, V, r8, code, grads, _stream())
        _lib.check(st, "mlora_linear_cross_entropy_backward")
    if da is not None and r8 != r:
        da, db = da[:r].contiguous(), db[:, :r].contiguous()
    return dx, da, db, dw


# ------------------------------------------------------- token embedding --

def _table_index(indices: torch.Tensor) -> torch.Tensor:
    """The indices in a row of int64."""
    if indices.dtype != torch.int64:
        if indices.dtype != torch.int32:
            raise ShapeError(f"indices must be int64 or int32, got {indices.dtype}")
        indices = indices.to(torch.int64)
    return indices.contiguous()


def embedding_run(indices: torch.Tensor, table: torch.Tensor, scale: float):
    """``embedding_fwd``'s output, its indices as the kernels take them, (T, V, D, scale)
    and the type's code: what its backward takes besides dy."""
    _need_here(table, indices)
    code = _dtype_code(table)
    if table.dim() != 2:
        raise ShapeError(f"the table must be [V, D], got {tuple(table.shape)}")
    V, D = table.shape
    idx = _table_index(indices)
    T = idx.numel()
    table = table.contiguous()
    out = table.new_empty((*idx.shape, D))
    if T and D:
        st = _lib.load().mlora_embedding_forward(idx.data_ptr(), table.data_ptr(), out.data_ptr(), T, V,
                                                 D, scale, code, _stream())
        if st:
            _lib.check(st, "mlora_embedding_forward")
    return out, idx, (T, V, D, scale), code


def embedding_fwd(indices: torch.Tensor, table: torch.Tensor, scale: float = 1.0) -> torch.Tensor:
    """scale * table[idx] for every index, [*indices.shape, D] (bf16, fp16 or fp32); an
    index outside the table gives a zero row and device status 0x107."""
    return embedding_run(indices, table, float(scale))[0]


def embedding_bwd(dy: torch.Tensor, indices: torch.Tensor, num_embeddings: int, scale: float = 1.0,
                  padding_idx: int | None = None) -> torch.Tensor:
    """The table's gradient [num_embeddings, D] in dy's dtype: scale times the sum of
    dy over each entry's tokens, in fp32 and in token order (the same bits in every
    run); zero for ``padding_idx``."""
    _need_here(dy, indices)
    idx = _table_index(indices)
    if dy.shape[:-1] != idx.shape:
        raise ShapeError(f"grad_output {tuple(dy.shape)} does not match indices {tuple(idx.shape)}")
    T, V, D = idx.numel(), int(num_embeddings), dy.shape[-1]
    code = _dtype_code(dy)
    dy = dy.contiguous()
    grad = dy.new_empty((V, D))
    if T == 0 or D == 0:
        return grad.zero_()
    nbytes = _lib.load().mlora_embedding_backward_workspace_bytes(T, D)
    ws = dy.new_empty(nbytes, dtype=torch.uint8)
    st = _lib.load().mlora_embedding_backward(idx.data_ptr(), dy.data_ptr(), grad.data_ptr(), T, V, D,
                                              float(scale), -1 if padding_idx is None else padding_idx,
                                              code, ws.data_ptr(), nbytes, _stream())
    _lib.check(st, "mlora_embedding_backward")
    return grad


# ---------------------------------------------------------------- dropout --

_U64 = 2 ** 64 - 1


def _drop_threshold(p: float) -> int:
    """Of 65536: p to the nearest multiple of 2^-16."""
    if not 0.0 <= p <= 1.0:
        raise ConfigurationError(f"dropout must be in [0, 1], got {p}")
    return round(65536 * p)


def _drop_seed(seed) -> tuple[int, int | None]:
    """(seed, device address or None) of an int, or of a CUDA int64 tensor of one element."""
    if torch.is_tensor(seed):
        _need_here(seed)
        if seed.dtype != torch.int64 or seed.numel() != 1:
            raise ShapeError("a seed tensor holds one int64")
        return 0, seed.data_ptr()
    return int(seed) & _U64, None


def dropout_plan(x: torch.Tensor, p: float, seed, call: int = 0, scaled: bool = True) -> tuple:
    """What ``dropout_run`` takes besides a tensor like x: all that is checked once for
    the forward and its backward.  (A seed tensor has to outlive both.)"""
    t = _drop_threshold(p)
    _need_here(x)
    s, s_dev = _drop_seed(seed)
    return (x.numel(), t, scaled, s, s_dev, call & _U64, _dtype_code(x))


def dropout_run(x: torch.Tensor, plan: tuple) -> torch.Tensor:
    """The dropout of a tensor of the plan's size, type and device."""
    if not x.is_contiguous():
        x = x.contiguous()
    out = torch.empty_like(x)
    if plan[0]:
        st = _lib.load().mlora_dropout(x.data_ptr(), out.data_ptr(), *plan, _stream())
        if st:
            _lib.check(st, "mlora_dropout")
    return out


def dropout(x: torch.Tensor, p: float, seed, call: int = 0, scaled: bool = True) -> torch.Tensor:
    """x with every element dropped (0) or scaled by the counter-based mask of ``seed``
    and ``call`` (see ``ops.dropout``); its gradient is the same call on dy.  Without
    ``scaled`` the kept elements are as they were."""
    return dropout_run(x, dropout_plan(x, p, seed, call, scaled))


def lora_linear_dropout_fwd(x2d: torch.Tensor, w0: torch.Tensor, a: torch.Tensor, b: torch.Tensor,
                            alpha: float, p: float, seed, call: int = 0):
    """(y, saved_xa) of y = x.W0^T + dropout((alpha/r).(x.A^T).B^T) for 2-D x [M, K], bf16
    or fp16; the mask as in ``dropout``, over [M, N]."""
    t = _drop_threshold(p)
    _need_here(x2d, w0, a, b)
    dt = x2d.dtype
    if dt not in (torch.bfloat16, torch.float16):
        raise ShapeError("counter-based LoRA dropout takes bf16 or fp16 activations")
    M, K = x2d.shape
    N = w0.shape[0]
    a, b, alpha, r = _pad_rank(a, b, alpha)
    _check_2d("W0", w0, (N, K), dt)
    _check_2d("A", a, (r, K), dt)
    _check_2d("B", b, (N, r), dt)
    s, s_dev = _drop_seed(seed)
    x2d, w0, a, b = (v.contiguous() for v in (x2d, w0, a, b))
    y = x2d.new_empty((M, N))
    saved = x2d.new_empty((rank_tile(r), (M + 7) // 8 * 8))
    if M == 0:
        return y, saved
    lib = _lib.load()
    ws = _workspace(lib.mlora_lora_forward_dropout_workspace_bytes(M, K, N, r, _DT[dt]), x2d.device)
    st = lib.mlora_lora_forward_dropout(_ptr(x2d), _ptr(w0), _ptr(a), _ptr(b), _ptr(y), _ptr(saved),
                                        M, K, N, r, float(alpha), t, s, s_dev,
                                        call & _U64, _DT[dt], _ptr(ws), ws.numel(),
                                        _stream())
    _lib.check(st, "mlora_lora_forward_dropout")
    return y, saved


def lora_linear_dropout_bwd(dy2d: torch.Tensor, x2d: torch.Tensor, w0: torch.Tensor, a: torch.Tensor,
                            b: torch.Tensor, alpha: float, saved_xa: torch.Tensor, p: float, seed,
                            call: int = 0, need_dx: bool = True,
                            da_out: torch.Tensor | None = None, db_out: torch.Tensor | None = None,
                            accumulate: bool = True, grad_dtype: torch.dtype | None = None,
                            on_grads=None):
    """(dx, dA, dB) of ``lora_linear_dropout_fwd``: the LoRA products take dropout(dy), the
    base's takes dy.  The other arguments as for ``lora_linear_bwd``; ``on_grads`` is
    called between dA/dB and the dx GEMM."""
    dz = dropout(dy2d, p, seed, call, scaled=False)  # exact: alpha takes the factor
    t = _drop_threshold(p)
    alpha = alpha * (65536 / (65536 - t) if t < 65536 else 0.0)
    dy2d = dy2d.contiguous()
    M, K = x2d.shape
    if not need_dx or M == 0:
        dx, da, db = lora_linear_bwd(dz, x2d, w0 if need_dx else None, a, b, alpha, saved_xa, 0.0,
                                     need_dx=need_dx, da_out=da_out, db_out=db_out,
                                     accumulate=accumulate, grad_dtype=grad_dtype)
        if on_grads is not None:
            on_grads()
        return dx, da, db
    dt = x2d.dtype
    N, r_orig = dy2d.shape[1], a.shape[0]
    a_p, b_p, alpha_p, r = _pad_rank(a, b, alpha)
    _check_2d("grad_output", dy2d, (M, N), dt)
    _check_saved(saved_xa, r, M, dt)
    x2d, w0, a_p, b_p = (v.contiguous() for v in (x2d, w0, a_p, b_p))
    into = da_out is not None or db_out is not None
    flags = 0
    if into:
        _check_grad_out(da_out, db_out, r, r_orig, K, N)
        da, db = da_out, db_out
        flags = _lib.BWD_ACCUMULATE if accumulate else 0
    elif grad_dtype == dt:
        flags = _lib.BWD_GRADS_16BIT
        da, db = dy2d.new_empty((r, K)), dy2d.new_empty((N, r))
    else:
        da = dy2d.new_empty((r, K), dtype=torch.float32)
        db = dy2d.new_empty((N, r), dtype=torch.float32)
    dx = dy2d.new_empty((M, K))
    lib = _lib.load()
    ws = dy2d.new_empty(_bwd_ws_bytes(M, K, N, r, _DT[dt]), dtype=torch.uint8)
    for phase, g in ((_lib.BWD_DEFER_DX, dz), (_lib.BWD_DX_ONLY, dy2d)):
        st = lib.mlora_lora_backward_ex(_ptr(g), _ptr(x2d), _ptr(w0), _ptr(a_p), _ptr(b_p),
                                        _ptr(saved_xa), _ptr(dx), _ptr(da), _ptr(db), M, K, N, r,
                                        float(alpha_p), 0.0, _DT[dt], flags | phase, _ptr(ws),
                                        ws.numel(), _stream())
        _lib.check(st, "mlora_lora_backward_ex")
        if phase == _lib.BWD_DEFER_DX and on_grads is not None:
            on_grads()
    if not into and r != r_orig:
        da, db = da[:r_orig].contiguous(), db[:, :r_orig].contiguous()
    return dx, da, db
