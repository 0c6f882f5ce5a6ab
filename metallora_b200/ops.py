"""LoRA operations (reference: python/metal_lora/ops.py), on sm_100a kernels.

Same function names, arguments and defaults as the reference so callers can
switch imports.  ``use_metal``/``kernel_kwargs`` are accepted and ignored: there
is exactly one implementation, the CUDA one, and no fallback.  All tensors must
be CUDA tensors; bf16, fp16 or fp32 (fp32 runs as split-precision bf16
tensor-core GEMMs, see ``kernels``).
"""
from __future__ import annotations

import torch
from torch.autograd import forward_ad

from . import _lib
from . import kernels as _k
from .exceptions import ConfigurationError, ShapeError
from .quant import ActivationCheckpoint, empty_checkpoint


def _checkpoint(x2d, checkpoint):
    """(checkpoint of ``x2d`` or None, whether the forward has to fill it):
    ``checkpoint`` is None, "mxint8", or one the caller made of the same x."""
    if checkpoint is None:
        return None, False
    if x2d.dtype not in (torch.bfloat16, torch.float16):
        raise ConfigurationError("activation checkpoints take bf16 or fp16 activations")
    if isinstance(checkpoint, ActivationCheckpoint):
        checkpoint.check()
        if checkpoint.rows != x2d.shape[0] or checkpoint.shape[-1] != x2d.shape[1] or \
                checkpoint.dtype != x2d.dtype or checkpoint.device != x2d.device:
            raise ShapeError(f"the checkpoint is of {tuple(checkpoint.shape)} {checkpoint.dtype} on "
                             f"{checkpoint.device}, x is {tuple(x2d.shape)} {x2d.dtype} on "
                             f"{x2d.device}")
        return checkpoint, False
    if checkpoint != "mxint8":
        raise ConfigurationError(f"unknown activation checkpoint {checkpoint!r}; use 'mxint8' or "
                                 "an ActivationCheckpoint")
    _k._need_cuda(x2d)
    return empty_checkpoint(x2d), True


def _keep_x(ctx, x2d, ckpt) -> tuple:
    """What the forward saves of x: (x, None), or the checkpoint's codes and
    scales (rebuilt by ``_kept_x``)."""
    ctx.x_meta = None if ckpt is None else (tuple(x2d.shape), x2d.dtype)
    return (x2d, None) if ckpt is None else (ckpt.codes, ckpt.scales)


def _kept_x(ctx, x2d, scales):
    if ctx.x_meta is None:
        return x2d
    ckpt = ActivationCheckpoint(x2d, scales, *ctx.x_meta)
    if x2d.stride(0) % 16:  # a saved-tensor hook (offloading) gave it back without its row gaps
        ckpt.codes = empty_checkpoint(x2d).codes.copy_(x2d)
    return ckpt


def _cast_ab(a, b, dtype):
    """A and B in ``dtype`` (``Tensor.to`` costs about 1 us where it changes nothing)."""
    return (a if a.dtype == dtype else a.to(dtype)), (b if b.dtype == dtype else b.to(dtype))


def _sink_accumulates(sink) -> bool:
    return sink is None or len(sink) < 3 or bool(sink[2])


class _LoRALinearFn(torch.autograd.Function):
    """y = x.W0^T + s.(x.A^T).B^T with the fused backward (dx, dA, dB in one
    launch sequence).  W0 gets a gradient only when it requires one (the
    reference freezes it by default, layers.py:77-78).

    A/B may be kept in a wider dtype than x (fp32 master factors with bf16
    compute): they are cast for the kernels and their gradients returned in
    their own dtype.  ``compute`` optionally supplies ready-made casts, and
    ``sink`` = (gA, gB) fp32 buffers receives the LoRA gradients by in-kernel
    accumulation instead of autograd (the trainer's flat gradient buffer);
    (gA, gB, False) writes them over the buffers' contents instead.  A fourth
    element ``on_grads`` (a callable) is called once dA/dB are enqueued and
    before the dx GEMM is: work it starts on another stream (a gradient
    exchange) overlaps that GEMM."""

    @staticmethod
    def forward(ctx, x2d, w0, a, b, alpha, compute, sink, checkpoint=None):
        a_c, b_c = compute if compute is not None else _cast_ab(a, b, x2d.dtype)
        ckpt, fill = _checkpoint(x2d, checkpoint)
        y, saved = _k.lora_linear_fwd(x2d, w0, a_c, b_c, alpha, save_xa=True,
                                      ckpt_out=ckpt if fill else None)
        ctx.save_for_backward(*_keep_x(ctx, x2d, ckpt), w0, a_c, b_c, saved)
        ctx.alpha = alpha
        ctx.sink = sink
        ctx.ab_dtypes = (a.dtype, b.dtype)
        return y

    @staticmethod
    def backward(ctx, dy):
        x2d, scales, w0, a_c, b_c, saved = ctx.saved_tensors
        x2d = _kept_x(ctx, x2d, scales)
        need_dx = ctx.needs_input_grad[0]
        sink = ctx.sink
        on_grads = sink[3] if sink is not None and len(sink) > 3 else None
        if on_grads is not None and need_dx and x2d.dtype != torch.float32:
            finish = _k.lora_linear_bwd_split(dy.contiguous(), x2d, w0, a_c, b_c, ctx.alpha,
                                              saved, sink[0], sink[1],
                                              accumulate=_sink_accumulates(sink))
            on_grads()
            dx, da, db = finish(), sink[0], sink[1]
        else:
            same = ctx.ab_dtypes[0] == ctx.ab_dtypes[1] == x2d.dtype  # 16-bit grads direct
            dx, da, db = _k.lora_linear_bwd(dy.contiguous(), x2d, w0 if need_dx else None, a_c,
                                            b_c, ctx.alpha, saved, 0.0, need_dx=need_dx,
                                            da_out=sink[0] if sink else None,
                                            db_out=sink[1] if sink else None,
                                            accumulate=_sink_accumulates(sink),
                                            grad_dtype=x2d.dtype if same else None)
            if on_grads is not None:
                on_grads()
        dw0 = None
        if ctx.needs_input_grad[1]:
            # trainable base weight (freeze_base=False): plain library GEMM
            dw0 = (dy.t().float() @ x2d.float()).to(w0.dtype)
        if dx is not None and not need_dx:
            dx = None
        if sink is not None:
            return dx, dw0, None, None, None, None, None, None
        da = da.to(ctx.ab_dtypes[0]) if ctx.needs_input_grad[2] else None
        db = db.to(ctx.ab_dtypes[1]) if ctx.needs_input_grad[3] else None
        return dx, dw0, da, db, None, None, None, None


_once = torch.autograd.function.once_differentiable


def _keep_seed(ctx, seed, *tensors):
    """Saves the tensors, and the seed aside or, a tensor itself, with them: its being
    written over before the backward is then noticed."""
    ctx.seed = None if torch.is_tensor(seed) else seed
    ctx.save_for_backward(*tensors, *(() if ctx.seed is not None else (seed,)))


def _kept_seed(ctx):
    """(the seed, the tensors saved with it)."""
    saved = ctx.saved_tensors
    return (saved[-1], saved[:-1]) if ctx.seed is None else (ctx.seed, saved)


class _LoRADropoutFn(torch.autograd.Function):
    """The LoRA linear with counter-based dropout on its LoRA term; W0 is frozen.
    ``compute`` and ``sink`` as in _LoRALinearFn."""

    @staticmethod
    def forward(ctx, x2d, w0, a, b, alpha, p, seed, call, compute, sink):
        a_c, b_c = compute if compute is not None else _cast_ab(a, b, x2d.dtype)
        y, saved = _k.lora_linear_dropout_fwd(x2d, w0, a_c, b_c, alpha, p, seed, call)
        _keep_seed(ctx, seed, x2d, w0, a_c, b_c, saved)
        ctx.plan = (alpha, p, call)
        ctx.sink = sink
        ctx.ab_dtypes = (a.dtype, b.dtype)
        return y

    @staticmethod
    @_once
    def backward(ctx, dy):
        seed, (x2d, w0, a_c, b_c, saved) = _kept_seed(ctx)
        alpha, p, call = ctx.plan
        sink = ctx.sink
        same = ctx.ab_dtypes[0] == ctx.ab_dtypes[1] == x2d.dtype
        need = ctx.needs_input_grad
        dx, da, db = _k.lora_linear_dropout_bwd(
            dy, x2d, w0, a_c, b_c, alpha, saved, p, seed, call,
            need_dx=need[0], da_out=sink[0] if sink else None, db_out=sink[1] if sink else None,
            accumulate=_sink_accumulates(sink), grad_dtype=x2d.dtype if same else None,
            on_grads=sink[3] if sink is not None and len(sink) > 3 else None)
        if sink is not None:
            return dx, *(None,) * 9
        da = da.to(ctx.ab_dtypes[0]) if need[2] else None
        db = db.to(ctx.ab_dtypes[1]) if need[3] else None
        return dx, None, da, db, *(None,) * 6


class _QLoRALinearFn(torch.autograd.Function):
    """The LoRA linear over a frozen quantised base (QLoRA): no gradient for
    the base; A/B handled as in _LoRALinearFn."""

    @staticmethod
    def forward(ctx, x2d, a, b, qw, alpha, compute, sink, checkpoint=None):
        a_c, b_c = compute if compute is not None else _cast_ab(a, b, x2d.dtype)
        ckpt, fill = _checkpoint(x2d, checkpoint)
        y, saved = _k.qlora_linear_fwd(x2d, qw, a_c, b_c, alpha, save_xa=True,
                                       ckpt_out=ckpt if fill else None)
        ctx.save_for_backward(*_keep_x(ctx, x2d, ckpt), a_c, b_c, saved)
        ctx.qw, ctx.alpha, ctx.sink = qw, alpha, sink
        ctx.ab_dtypes = (a.dtype, b.dtype)
        return y

    @staticmethod
    def backward(ctx, dy):
        x2d, scales, a_c, b_c, saved = ctx.saved_tensors
        x2d = _kept_x(ctx, x2d, scales)
        sink = ctx.sink
        need_dx = ctx.needs_input_grad[0]
        # 16-bit gradients straight from the kernel where no cast would follow
        same = ctx.qw.scheme == "mxfp4" and ctx.ab_dtypes[0] == ctx.ab_dtypes[1] == x2d.dtype
        dx, da, db = _k.qlora_linear_bwd(dy.contiguous(), x2d, ctx.qw, a_c, b_c, ctx.alpha, saved,
                                         0.0, need_dx=need_dx,
                                         da_out=sink[0] if sink else None,
                                         db_out=sink[1] if sink else None,
                                         accumulate=_sink_accumulates(sink),
                                         grad_dtype=x2d.dtype if same else None)
        if sink is not None and len(sink) > 3 and sink[3] is not None:
            sink[3]()
        if sink is not None:
            return dx, None, None, None, None, None, None, None
        if not same:
            da, db = da.to(ctx.ab_dtypes[0]), db.to(ctx.ab_dtypes[1])
        return (dx, da if ctx.needs_input_grad[1] else None,
                db if ctx.needs_input_grad[2] else None, None, None, None, None, None)


def _forward_mode() -> bool:
    """Whether a forward-mode level is open (if that cannot be told: True)."""
    return getattr(forward_ad, "_current_level", 0) >= 0


def qlora_forward(x, qweight, A, B, alpha: float = 16.0, _compute=None, _sink=None,  # noqa: N803
                  checkpoint=None):
    """LoRA forward over a quantised base (``quant.QuantizedWeight``):
    ``x.deq(W)^T + (alpha/rank).(x.A^T).B^T`` with the dequantisation fused
    into the GEMM (replaces qlora_forward_nf4/int4, lora_quantized.metal:29-164).
    An MXFP4 base multiplies x rounded to MXFP4 (the gradient passes straight
    through that rounding).  ``checkpoint`` as for ``lora_forward``."""
    shp = x.shape
    x2d = x if len(shp) == 2 else x.reshape(-1, shp[-1])
    grad = torch.is_grad_enabled() and (x.requires_grad or A.requires_grad or B.requires_grad)
    # the short path has no place for a forward-mode tangent, which no_grad does not
    # switch off (the function below refuses one)
    if qweight.scheme == "mxfp4" and checkpoint is None and not grad and not _forward_mode():
        a, b = _compute if _compute is not None else _cast_ab(A, B, x.dtype)
        out = _k.qlora_linear_fwd(x2d, qweight, a, b, float(alpha))[0]
    else:
        out = _QLoRALinearFn.apply(x2d, A, B, qweight, float(alpha), _compute, _sink, checkpoint)
    return out if len(shp) == 2 else out.reshape(*shp[:-1], qweight.shape[0])


def _apply(x2d, W0, A, B, alpha, compute=None, sink=None, checkpoint=None):
    return _LoRALinearFn.apply(x2d, W0, A, B, float(alpha), compute, sink, checkpoint)


def lora_forward(x, W0, A, B, alpha: float = 16.0, dropout: float = 0.0,  # noqa: N803
                 training: bool = False, use_metal: bool = True, kernel_kwargs: dict | None = None,
                 _compute=None, _sink=None, checkpoint=None, dropout_seed=None,
                 dropout_call: int = 0):
    """LoRA forward ``h = x.W0^T + (alpha/rank).(x.A^T).B^T`` (ops.py:32-103).

    x is [batch, seq, in] or [seq, in] (any leading shape works); rank is read
    from ``B.shape[1]`` (ops.py:73).  With ``training`` and ``dropout > 0`` the
    dropout mask multiplies the LoRA term only, as at ops.py:96-98.

    ``checkpoint`` keeps x for the backward in 8 bits instead of 16: "mxint8"
    quantises it here, a ``quant.ActivationCheckpoint`` of x is used as it is
    (layers that share an input share one).  dA then comes from the
    checkpoint's values; y does not change, and dx and dB at most in the order
    of their fp32 sums.  It needs a frozen W0 and no dropout, which read x
    itself.

    ``dropout_seed`` (an int, or a CUDA int64 tensor of one element) takes the mask
    from the counter-based generator of ``dropout`` instead of torch's: it is
    made again in the backward and never stored, and the call runs on the fused
    kernels.  ``dropout_call`` numbers the uses of one seed.  It needs a frozen W0,
    bf16 or fp16, and out_features in multiples of 8.
    """
    if x.shape[-1] != W0.shape[1]:
        raise ShapeError(f"x last dim {x.shape[-1]} != in_features {W0.shape[1]}")
    shp = x.shape
    x2d = x.reshape(-1, shp[-1])
    if checkpoint is not None and (W0.requires_grad or (training and dropout > 0)):
        raise ConfigurationError("an activation checkpoint needs a frozen W0 and no dropout")
    if training and dropout > 0 and dropout_seed is not None:
        if W0.requires_grad:
            raise ConfigurationError("counter-based LoRA dropout needs a frozen W0")
        out = _LoRADropoutFn.apply(x2d, W0, A, B, float(alpha), float(dropout), dropout_seed,
                                   int(dropout_call), _compute, _sink)
    elif training and dropout > 0:
        # ops.py:96-98: output = w0x + scale * bax * mask / (1 - dropout)
        zero_b = torch.zeros_like(B)
        w0x = _apply(x2d, W0, A, zero_b, alpha)
        scale = alpha / B.shape[1]
        bax = (x2d @ A.t()) @ B.t()
        mask = torch.bernoulli(torch.full_like(bax, 1.0 - dropout))
        out = w0x + scale * bax * mask / (1.0 - dropout)
    else:
        out = _apply(x2d, W0, A, B, alpha, _compute, _sink, checkpoint)
    return out.reshape(*shp[:-1], W0.shape[0])


def lora_forward_inference(x, w_merged):
    """Merged-weight forward (ops.py:106-114): ``x.W'^T`` with no adapter."""
    shp = x.shape
    y = _k.linear(x.reshape(-1, shp[-1]), w_merged)
    return y.reshape(*shp[:-1], w_merged.shape[0])


def lora_backward(grad_output, x, A, B, alpha: float = 16.0, clip_value: float = 1.0,  # noqa: N803
                  use_metal: bool = True, saved_xa=None):
    """Gradients of A and B (ops.py:117-155), clipped elementwise to
    +-clip_value after the full reduction, returned in A's/B's dtype.

    x may be an 8-bit ``quant.ActivationCheckpoint``: dA is taken from its
    values, and dB from ``saved_xa``, the (alpha/rank) x.A^T that the forward
    kept (``kernels.lora_linear_fwd(..., save_xa=True)``), or without it from
    the checkpoint's values too."""
    g = grad_output
    if g.dim() != 2:
        g = g.reshape(-1, g.shape[-1])
    if not torch.is_tensor(x):
        clip = float(clip_value) if clip_value is not None else 0.0
        if saved_xa is None:
            x = x.dequantize().reshape(-1, x.shape[-1])
        _, da, db = _k.lora_linear_bwd(g, x, None, A, B, alpha, saved_xa, clip, need_dx=False,
                                       grad_dtype=A.dtype if A.dtype == B.dtype else None)
        return (da if da.dtype == A.dtype else da.to(A.dtype),
                db if db.dtype == B.dtype else db.to(B.dtype))
    xx = x.reshape(-1, x.shape[-1])
    clip = float(clip_value) if clip_value is not None else 0.0
    _, da, db = _k.lora_linear_bwd(g, xx, None, A, B, alpha, saved_xa, clip, need_dx=False)
    return da.to(A.dtype), db.to(B.dtype)


# ops.py:158-159
lora_backward_efficient = lora_backward


def merge_lora_weights(W0, A, B, alpha: float = 16.0):  # noqa: N803
    """``W0 + (alpha/A.shape[0]) . B.A`` (ops.py:162-172) on the merge kernel."""
    return _k.merge(W0, A, B, alpha)


def unmerge_lora_weights(w_merged, W0, A, B, alpha: float = 16.0):  # noqa: N803
    """Recovers (A, B) from merged weights by truncated SVD (ops.py:175-193).
    Not on the hot path: uses torch.linalg.svd."""
    rank = A.shape[0]
    scale = alpha / rank
    delta = (w_merged.float() - W0.float()) / scale
    u, s, vt = torch.linalg.svd(delta, full_matrices=False)
    sqrt_s = torch.sqrt(s[:rank])
    a_rec = torch.diag(sqrt_s) @ vt[:rank, :]
    b_rec = u[:, :rank] @ torch.diag(sqrt_s)
    return a_rec.to(A.dtype), b_rec.to(B.dtype)


def multi_adapter_forward(x, W0, adapters_A, adapters_B, adapter_ids, alpha: float = 16.0):  # noqa: N803
    """Per-sample adapters over a shared base (the ``lora_multi_adapter`` kernel,
    kernels/lora_kernels.metal:440-508): ``y[b] = x[b].W0^T + (alpha/r)
    (x[b].A_id^T).B_id^T`` with ``id = adapter_ids[b]``.

    x [B, S, K]; W0 [N, K] or None (LoRA term only); adapters_A [n, r, K];
    adapters_B [n, N, r]; adapter_ids: ints, one per sample.  Only the
    adapters the batch uses are stacked; more than fit one launch
    (n * r <= 256) are applied in groups.
    """
    if x.dim() == 2:
        x = x.unsqueeze(0)
    Bsz, S, K = x.shape
    n_all, r, _ = adapters_A.shape
    N = adapters_B.shape[1]
    # ids are small host data: grouping and per-token ids are built on the host
    # (a CUDA tensor of ids is read back once)
    ids = [int(i) for i in (adapter_ids.tolist() if torch.is_tensor(adapter_ids) else adapter_ids)]
    if len(ids) != Bsz:
        raise ShapeError(f"{len(ids)} adapter ids for {Bsz} samples")
    if any(i < 0 or i >= n_all for i in ids):
        raise ShapeError(f"adapter ids must be in [0, {n_all})")
    x2d = x.reshape(-1, K)
    used = sorted(set(ids))
    r8 = (r + 7) // 8 * 8
    per = max(1, _k.MAX_STACKED_RANK // r8)
    y = None
    for g0 in range(0, len(used), per):
        group = used[g0:g0 + per]
        sel = torch.tensor(group, dtype=torch.int64).to(x.device, non_blocking=True)
        a, b = adapters_A.index_select(0, sel).to(x.dtype), adapters_B.index_select(0, sel).to(x.dtype)
        if r8 != r:  # zero-padded rank, alpha/r unchanged
            a = torch.nn.functional.pad(a, (0, 0, 0, r8 - r))
            b = torch.nn.functional.pad(b, (0, r8 - r))
        a_stack = a.reshape(len(group) * r8, K)
        b_stack = b.permute(1, 0, 2).reshape(N, len(group) * r8)
        slot = {g: j for j, g in enumerate(group)}
        tok_host = torch.tensor([slot.get(i, -1) for i in ids], dtype=torch.int32)
        tok = tok_host.repeat_interleave(S).to(x.device, non_blocking=True)
        base = W0.to(x.dtype) if (W0 is not None and y is None) else None
        part = _k.multi_lora_fwd(x2d, base, a_stack, b_stack, tok, r8, float(alpha) * r8 / r)
        y = part if y is None else y + part
    return y.reshape(Bsz, S, N)


class _LinearCrossEntropyFn(torch.autograd.Function):
    """The gradients are made in the forward, where a piece's logits are at hand, up
    to the upstream factor, which the backward multiplies in (see
    ``linear_cross_entropy``).  ``compute`` and ``sink`` as in _LoRALinearFn."""

    @staticmethod
    def forward(ctx, x2d, w, a, b, labels, plan):
        alpha, ignore_index, reduction, compute, sink, grad_mode = plan
        # (what needs_input_grad says holds under no_grad too)
        need = ctx.needs_input_grad if grad_mode else (False,) * 4
        grads = (_lib.HEAD_GRAD_X if need[0] else 0) | (_lib.HEAD_GRAD_W if need[1] else 0)
        a_c = b_c = None
        if a is not None:
            a_c, b_c = compute if compute is not None else _cast_ab(a, b, x2d.dtype)
            if need[2] or need[3]:
                grads |= _lib.HEAD_GRAD_AB
                ctx.rank, ctx.ab_dtypes = a.shape[0], (a.dtype, b.dtype)
        loss, state = _k.linear_cross_entropy_fwd(x2d, w, labels, a_c, b_c, alpha, ignore_index,
                                                  reduction, grads)
        ctx.save_for_backward(state, w)
        ctx.plan = (x2d.shape[0], 0 if a is None else a.shape[0], reduction, grads)
        ctx.sink = sink
        return loss

    @staticmethod
    @_once
    def backward(ctx, grad):
        state, w = ctx.saved_tensors
        m, r, reduction, grads = ctx.plan
        sink = ctx.sink if grads & _lib.HEAD_GRAD_AB else None
        same = grads & _lib.HEAD_GRAD_AB and ctx.ab_dtypes[0] == ctx.ab_dtypes[1]
        dx, da, db, dw = _k.linear_cross_entropy_bwd(
            grad, state, w, m, r, reduction, grads, da_out=sink[0] if sink else None,
            db_out=sink[1] if sink else None, accumulate=_sink_accumulates(sink),
            ab_dtype=ctx.ab_dtypes[0] if same else torch.float32)
        if sink is not None:
            if len(sink) > 3 and sink[3] is not None:
                sink[3]()
            da = db = None
        elif da is not None and not same:
            da, db = da.to(ctx.ab_dtypes[0]), db.to(ctx.ab_dtypes[1])
        need = ctx.needs_input_grad
        return dx, dw, da if need[2] else None, db if need[3] else None, None, None


def linear_cross_entropy(x, weight, labels, A=None, B=None, alpha: float = 16.0,  # noqa: N803
                         ignore_index: int = -100, reduction: str = "mean",
                         _compute=None, _sink=None):
    """Softmax cross entropy of a linear head over a large vocabulary, from the hidden
    states: ``cross_entropy(x.weight^T [+ (alpha/r)(x.A^T).B^T], labels)`` without the
    [tokens, vocabulary] logits.  During the forward, and for gradients alone, 16 bits
    of each are held for as many tokens as fill 2 GiB (256 at least); a loss without
    gradients holds 8 bytes for each 96 to 128 of them.

    x [..., K] (bf16 or fp16), weight [V, K] of the same type, labels int [...];
    A [r, K] and B [V, r] (both or neither) are a LoRA head's factors.  Tokens
    labelled ``ignore_index`` have no loss and cost nothing; one whose label is
    outside [0, V) is left out too and reported in the device status (0x107).
    ``reduction`` is "mean" (over the counted tokens; NaN for none), "sum" or
    "none" (a loss per token, 0 where there is none); the result is fp32.

    Gradients reach x, A and B, and weight where it requires one.  They are made in
    the forward, with the logits; the backward scales them.  "none" takes
    gradients of x alone: those of weights need to know in the forward how the
    tokens are weighted.  K must be a multiple of 8, and V with A and B."""
    if reduction not in ("mean", "sum", "none"):
        raise ConfigurationError(f"unknown reduction {reduction!r}")
    if (A is None) != (B is None):
        raise ConfigurationError("a LoRA head needs both A and B")
    if x.shape[-1] != weight.shape[1]:
        raise ShapeError(f"x last dim {x.shape[-1]} != in_features {weight.shape[1]}")
    if labels.shape != x.shape[:-1]:
        raise ShapeError(f"labels {tuple(labels.shape)} do not match x {tuple(x.shape)}")
    if reduction == "none" and torch.is_grad_enabled() and \
            any(t is not None and t.requires_grad for t in (weight, A, B)):
        raise ConfigurationError("reduction='none' takes gradients of x alone; detach the head's "
                                 "weights or use 'mean' or 'sum'")
    flat = x.dim() == 2
    if A is None and not (weight.requires_grad and torch.is_grad_enabled()):  # a frozen head
        x2d = x if flat else x.reshape(-1, x.shape[-1])
        hang = _hang(x2d, weight)
        loss, state = _k.linear_cross_entropy_fwd(
            x2d, weight, labels if flat else labels.reshape(-1), None, None, 16.0, ignore_index,
            reduction, _lib.HEAD_GRAD_X if hang else 0)
        if hang:
            _lib.autograd().attach_linear_cross_entropy(loss, x2d, state, weight, x2d.shape[0],
                                                        reduction == "none", reduction == "mean",
                                                        _k._DT[x2d.dtype])
        return loss if flat or reduction != "none" else loss.reshape(labels.shape)
    loss = _LinearCrossEntropyFn.apply(x if flat else x.reshape(-1, x.shape[-1]), weight, A, B,
                                       labels if flat else labels.reshape(-1),
                                       (float(alpha), ignore_index, reduction, _compute, _sink,
                                        torch.is_grad_enabled()))
    return loss if flat or reduction != "none" else loss.reshape(labels.shape)


def _hang(x, *rest) -> bool:
    """Whether the output of an operator gets a backward node, for x's gradient.  (There
    is no forward-mode derivative: a tangent of x or the rest is refused.)"""
    if _forward_mode() and any(forward_ad.unpack_dual(t).tangent is not None for t in (x, *rest)):
        raise NotImplementedError("this operator has no forward-mode derivative")
    return x.requires_grad and torch.is_grad_enabled()


def dropout(x, p: float, seed, call: int = 0, training: bool = True):
    """Dropout whose mask is never stored: ``kept ? x * 65536 / (65536 - t) : 0`` with
    t = round(65536 p), a dropped element being 0 whatever it was.

    The mask is a function of ``seed`` (an int, or a CUDA int64 tensor of one element,
    which a replayed graph reads anew), ``call``, which numbers the uses of one seed,
    and the element's place in x (row-major): half-word e % 8, the low half first, of
    the four words that Philox4x32-10 (Salmon et al., 2011) makes of the key ``seed``
    and the 128-bit counter (e // 8, call); kept where it is at least t.  The backward
    makes it again.  Any shape; bf16, fp16 or fp32.  Without ``training`` x is returned
    as it is."""
    if not 0.0 <= p <= 1.0:
        raise ConfigurationError(f"dropout must be in [0, 1], got {p}")
    if not training:
        return x
    plan = _k.dropout_plan(x, p, seed, call)
    out = _k.dropout_run(x, plan)
    if _hang(x):
        n, t, scaled, value, _, use, code = plan
        _lib.autograd().attach_dropout(out, x, n, t, scaled, value, use, code,
                                       seed if torch.is_tensor(seed) else None)
    return out


def embedding(indices, table, scale: float = 1.0, padding_idx: int | None = None):
    """``scale * table[indices]`` [*indices.shape, D] for int indices into table [V, D]
    (bf16, fp16 or fp32), and the gradient of a trained table: scale times the sum of
    dy over each entry's tokens, in fp32, in token order, the same bits in every run.

    ``padding_idx`` (negative: from the end) has no gradient.  An index outside the
    table gives a zero row and no gradient, and is reported in the device status
    (0x107)."""
    if table.dim() != 2:
        raise ShapeError(f"the table must be [V, D], got {tuple(table.shape)}")
    if padding_idx is not None:
        rows = table.shape[0]
        if not -rows <= padding_idx < rows:
            raise ConfigurationError(f"padding_idx {padding_idx} is outside the table's {rows} rows")
        padding_idx = int(padding_idx) % rows
    out, idx, sizes, code = _k.embedding_run(indices, table, float(scale))
    if _hang(table):
        _lib.autograd().attach_embedding(out, table, idx, *sizes,
                                         -1 if padding_idx is None else padding_idx, code)
    return out
