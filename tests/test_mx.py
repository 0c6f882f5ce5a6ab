"""Microscaled formats: MXFP4 bases, MXINT8 activation checkpoints, their
product and gradients, against 64-bit restatements.

Tolerances: a rounding to a 16-bit type is off by at most half a step,
``h = eps / 2`` relative to the value (bf16 2^-8, fp16 2^-11), plus half of the
type's smallest subnormal step; an fp32 sum of n terms by at most ``n 2^-23``
of the sum of their magnitudes (each of the n additions rounds or truncates at
2^-23 of a partial sum, which that sum bounds).
"""
import ctypes as C

import numpy as np
import pytest
import torch

from metallora_b200 import _lib, kernels, ops, quant
from metallora_b200.exceptions import (ConfigurationError, DeviceError, MetalLoRAError,
                                       QuantizationError, ShapeError)
from metallora_b200.layers import LoRALinear
from metallora_b200.trainer import LoRATrainer, TrainingConfig
from oracle import mx_oracle

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
ACC = 2.0 ** -23


def _half_step(dt):
    return torch.finfo(dt).eps / 2


def _tiny(dt):
    """Half of the smallest subnormal step."""
    return {BF16: 2.0 ** -134, FP16: 2.0 ** -25}[dt]


def _np(t):
    return t.detach().double().cpu().numpy()


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _acts(rows, k, dt, seed=0):
    """Values of very different size, exact zeros, whole zero blocks."""
    g = _gen(seed)
    x = torch.randn((rows, k), generator=g) * torch.exp2(
        torch.randint(-6, 7, (rows, 1), generator=g).float())
    x[torch.rand((rows, k), generator=g) < 0.1] = 0
    if k >= 64:
        x[0, 32:64] = 0
    return x.to(dt)


def _edge_rows(dt):
    """One row of ties, saturation, signs, subnormals, extremes, infinity and
    NaN blocks: 32 features a block."""
    fi = torch.finfo(dt)
    t = [0.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, 7.75, -0.25, -0.75, -5.0, -7.75, -0.0,
         0.125, 0.375, 4.0, -4.0, 0.5, -0.5, 1.0, -1.0, 1.5, -1.5, 2.0, -2.0, 3.0, -3.0, 0.0625, -6.0]
    i8 = [127.5 / 64, -127.5 / 64, 1.0, -1.0, 0.5 / 64, 1.5 / 64, 2.5 / 64, -0.5 / 64, -1.5 / 64,
          126.5 / 64, -126.5 / 64, 0.0] + [i / 64 for i in range(20)]
    sub = [fi.smallest_normal / 2, -fi.smallest_normal / 4] + [0.0] * 30
    top = [fi.max, -fi.max] + [fi.max / 2 ** i for i in range(30)]
    inf = [float("inf")] + [1.0] * 31
    nan = [1.0, float("nan")] + [2.0] * 30
    small = [float(torch.tensor(fi.smallest_normal) * 3)] * 32
    one = [0.0] * 31 + [-1.0]
    return torch.tensor([t + i8 + sub + top + inf + nan + small + one]).to(dt)


def _mx_quant_scales(ckpt):
    """Scale bytes [M, ceil(K/32)] of a checkpoint."""
    M, K = ckpt.rows, ckpt.shape[-1]
    return ckpt.scales.permute(1, 0, 2).flatten(1)[:M, : -(-K // 32)].cpu().numpy()


# ------------------------------------------------------------------ refusals --

def test_scheme_refusals():
    w = torch.zeros(4, 64)
    for kw in ({"group": 64}, {"lean": True}):
        with pytest.raises(QuantizationError):
            quant.quantize(w, "mxfp4", **kw)
    with pytest.raises(DeviceError):
        quant.quantize(w, "mxfp4")
    with pytest.raises(DeviceError):
        quant.checkpoint_activation(w)
    codes, scales = torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 2, dtype=torch.uint8)
    ok = quant.from_reference_layout("mxfp4", codes, scales, None, (4, 64), 32)
    assert ok.nbytes() == 4 * 32 + 4 * 2
    for bad in ((codes, scales, None, (4, 64), 64), (codes[:3], scales, None, (4, 64), 32),
                (codes, scales.int(), None, (4, 64), 32), (codes, scales[:, :1], None, (4, 64), 32),
                (codes, scales, scales, (4, 64), 32)):
        with pytest.raises(QuantizationError):
            quant.from_reference_layout("mxfp4", *bad)


def _cpu_ckpt(M=6, K=40):
    codes = torch.zeros((M, 48), dtype=torch.int8)[:, :K]
    return quant.ActivationCheckpoint(codes, torch.zeros((1, 8, 4), dtype=torch.uint8), (M, K), BF16)


def test_checkpoint_layout_refusals():
    c = _cpu_ckpt()
    c.check()
    for change in ({"codes": c.codes.contiguous()}, {"codes": c.codes.to(torch.uint8)},
                   {"codes": c.codes[:5]}, {"scales": c.scales[:, :6]},
                   {"scales": c.scales.to(torch.int8)}, {"shape": (6, 41)},
                   {"scales": c.scales.transpose(1, 2).contiguous().transpose(1, 2)}):
        bad = quant.ActivationCheckpoint(**{**c.__dict__, **change})
        with pytest.raises(ShapeError):
            bad.check()
    with pytest.raises(DeviceError):
        c.dequantize()


def test_configuration_refusals():
    with pytest.raises(ConfigurationError):
        LoRALinear(64, 64, activation_checkpoint="fp8")
    with pytest.raises(ConfigurationError):
        LoRATrainer(torch.nn.Sequential(LoRALinear(64, 64)),
                    TrainingConfig(activation_checkpoint="int8"))
    x, w = torch.zeros(4, 64, dtype=BF16), torch.zeros(64, 64, dtype=BF16)
    a, b = torch.zeros(8, 64, dtype=BF16), torch.zeros(64, 8, dtype=BF16)
    with pytest.raises(ConfigurationError):  # dropout reads x itself
        ops.lora_forward(x, w, a, b, dropout=0.5, training=True, checkpoint="mxint8")
    with pytest.raises(ConfigurationError):  # so does a trainable base
        ops.lora_forward(x, w.clone().requires_grad_(), a, b, checkpoint="mxint8")
    for bad in ("fp8", _cpu_ckpt()):
        with pytest.raises(MetalLoRAError):
            ops._checkpoint(x, bad)
    with pytest.raises(ConfigurationError):
        ops._checkpoint(x.float(), "mxint8")


def test_c_abi_refusals():
    """Bad arguments are refused before any device call."""
    lib = _lib.load()
    buf = C.create_string_buffer(1 << 16)
    p = (C.addressof(buf) + 255) // 256 * 256
    mx = _lib.QUANT_MXFP4
    bad = _lib.MLORA_ERR_INVALID_ARG
    assert lib.mlora_quantize(p, 0, 4, 64, mx, 64, p, p, None, None) == bad
    assert b"group" in lib.mlora_last_error_message()
    assert lib.mlora_quantize(p, 0, 4, 63, mx, 32, p, p, None, None) == bad
    assert lib.mlora_quantize(p, 0, 0, 64, mx, 32, p, p, None, None) == bad
    assert lib.mlora_quantize(p, 0, 4, 64, mx, 32, p, p + 1, None, None) == bad
    assert lib.mlora_dequantize(mx, None, p, None, 4, 64, 32, p, 0, None) == bad
    assert lib.mlora_act_checkpoint(p, 0, 4, 40, p, 39, p, None) == bad
    assert lib.mlora_act_checkpoint(p, 3, 4, 40, p, 48, p, None) == bad
    assert lib.mlora_act_checkpoint(p, 0, 4, 40, p, 48, p + 2, None) == bad
    assert lib.mlora_act_restore(None, 48, p, 4, 40, p, 0, None) == bad
    assert lib.mlora_act_checkpoint_scales_bytes(5, 129) == 2 * 8 * 4
    assert lib.mlora_act_checkpoint_scales_bytes(0, 129) == 0

    def bwd(codes=p, ld=64, scales=p, saved=p, dtype=0, flags=0, dx=None, w0=None):
        return lib.mlora_lora_backward_ckpt(p, codes, ld, scales, w0, p, p, saved, dx, p, p, 4, 64, 64,
                                            8, 1.0, 0.0, dtype, flags, p, 1 << 12, None)
    for kw in ({"codes": None}, {"codes": p + 8}, {"scales": None}, {"scales": p + 4}, {"ld": 56},
               {"ld": 72}, {"saved": None}, {"flags": 16}, {"dx": p}, {"flags": 6}):
        assert bwd(**kw) == bad, kw
    assert bwd(dtype=2) != 0

    def qfwd(K=64, group=32, dtype=0, x=p):
        return lib.mlora_qlora_forward_ex(x, mx, p, p, None, p, group, p, p, p, None, 4, K, 64, 8, 1.0,
                                          dtype, p, 1 << 12, None)
    for kw in ({"K": 48}, {"group": 64}, {"dtype": 2}, {"x": None}, {"x": p + 2}):
        assert qfwd(**kw) in (bad, _lib.MLORA_ERR_UNSUPPORTED), kw
    staged = lib.mlora_qlora_backward_workspace_bytes(64, 256, 128, 8, mx, 32)
    assert staged >= 128 * 256 * 2
    assert lib.mlora_qlora_lean_workspace_bytes(64, 256, 128, 8, mx, 32, 1) < staged
    assert lib.mlora_qlora_prepared_scales_bytes(mx, 129, 160, 32) == 2 * 2 * 512


def test_other_devices_are_refused(monkeypatch):
    """Kernels launch on the current device; tensors of another one are refused."""
    class Stub:
        device = torch.device("cuda:1")

        @staticmethod
        def get_device():
            return 1
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    with pytest.raises(DeviceError, match="cuda:1"):
        kernels._need_current(Stub)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 1)
    kernels._need_current(Stub)


def test_pack_round_trip():
    g = _gen(3)
    codes = torch.randint(0, 256, (24, 48), generator=g, dtype=torch.uint8)
    scales = torch.randint(100, 140, (24, 3), generator=g, dtype=torch.uint8)
    qw = quant.from_reference_layout("mxfp4", codes, scales, None, (24, 96), 32)
    tensors, meta = quant.pack_quantized({"w": qw})
    got = quant.unpack_quantized(tensors, meta)["w"]
    assert got.scheme == "mxfp4" and got.group == 32 and got.shape == (24, 96) and got.zeros is None
    assert torch.equal(got.codes, codes) and torch.equal(got.scales, scales)
    tensors["w.scales"] = tensors["w.scales"].half()
    with pytest.raises(QuantizationError):
        quant.unpack_quantized(tensors, meta)


# ------------------------------------------------------------------- formats --

@pytest.mark.gpu
@pytest.mark.parametrize("dt", [BF16, FP16, FP32])
@pytest.mark.parametrize("rows,k", [(1, 2), (1, 32), (3, 34), (5, 40), (33, 96), (7, 250), (9, 1000),
                                    (130, 1056), (65, 4096)])
def test_mxfp4_quantize_exact(cuda, dt, rows, k):
    w = _acts(rows, k, dt, seed=k)
    qw = quant.quantize(w.to(cuda), "mxfp4")
    val, byte = mx_oracle.mxfp4(_np(w))
    np.testing.assert_array_equal(qw.scales.cpu().numpy(), byte)
    # the product's table: 512-byte blocks of 128 rows x 4 scale bytes
    tab = qw._prepared.view(-(-rows // 128), -(-k // 128), 32, 4, 4).permute(0, 3, 2, 1, 4)
    tab = tab.reshape(-(-rows // 128) * 128, -1).cpu().numpy()
    np.testing.assert_array_equal(tab[:rows, : byte.shape[1]], byte)
    assert not tab[:rows, byte.shape[1]:].any()
    np.testing.assert_array_equal(mx_oracle.unpack_fp4(qw.codes.cpu().numpy(), byte), val)
    for out in (FP32, BF16):
        np.testing.assert_array_equal(_np(qw.dequantize(out)), val)
    np.testing.assert_array_equal(_np(qw.dequantize(FP16)),
                                  _np(torch.from_numpy(val).to(FP16)))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [BF16, FP16, FP32])
@pytest.mark.parametrize("shape", [(1, 1), (1, 8), (3, 33), (5, 40), (33, 96), (7, 250), (9, 1000),
                                   (2, 65, 1056), (65, 4096), (4, 0, 64)])
def test_mxint8_checkpoint_exact(cuda, dt, shape):
    rows = int(np.prod(shape[:-1]))
    x = _acts(rows, shape[-1], dt, seed=shape[-1]) if rows else torch.zeros(0, shape[-1], dtype=dt)
    c = quant.checkpoint_activation(x.reshape(shape).to(cuda))
    c.check()
    assert c.shape == shape and c.dtype == dt and c.rows == rows
    assert c.dequantize().shape == shape
    if not rows:
        return
    val, codes, byte = mx_oracle.mxint8(_np(x))
    np.testing.assert_array_equal(c.codes.cpu().numpy(), codes)
    np.testing.assert_array_equal(_mx_quant_scales(c), byte)
    for out in (FP32, BF16):
        np.testing.assert_array_equal(_np(c.dequantize(out)).reshape(rows, -1), val)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [BF16, FP16, FP32])
@pytest.mark.parametrize("cut", [0, 1])
def test_edge_values_exact(cuda, dt, cut):
    """Ties, saturation, subnormals, extremes, infinities and NaN, through the
    vector path and (odd row length) the element path."""
    x = _edge_rows(dt)
    if cut:
        x = torch.cat([x, x], 1)[:, : x.shape[1] + 2]
    val, byte = mx_oracle.mxfp4(_np(x))
    qw = quant.quantize(x.to(cuda), "mxfp4")
    np.testing.assert_array_equal(qw.scales.cpu().numpy(), byte)
    np.testing.assert_array_equal(_np(qw.dequantize(FP32)), val)
    val, codes, byte = mx_oracle.mxint8(_np(x))
    c = quant.checkpoint_activation(x.to(cuda))
    np.testing.assert_array_equal(_mx_quant_scales(c), byte)
    np.testing.assert_array_equal(c.codes.cpu().numpy(), codes)
    np.testing.assert_array_equal(_np(c.dequantize(FP32)), val)
    np.testing.assert_array_equal(_np(c.dequantize(BF16)), val)


@pytest.mark.gpu
def test_quantize_strided_and_unaligned(cuda):
    """Transposed, sliced and offset inputs give the codes of their contiguous copy."""
    base = torch.randn(200, 264, generator=_gen(1)).to(BF16).to(cuda)
    for v in (base.t(), base[::3, 5:101], base.flatten()[3:3 + 64 * 96].view(64, 96)):
        a, b = quant.quantize(v, "mxfp4"), quant.quantize(v.clone().contiguous(), "mxfp4")
        assert torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales)
        ca, cb = quant.checkpoint_activation(v), quant.checkpoint_activation(v.clone().contiguous())
        assert torch.equal(ca.codes, cb.codes) and torch.equal(ca.dequantize(), cb.dequantize())


# ------------------------------------------------------------------- product --

def _fwd_inputs(M, K, N, r, dt, cuda, seed=0):
    g = _gen(seed + 7 * M + K + N + r)
    x = _acts(M, K, dt, seed=seed + 1)
    w = (torch.randn(N, K, generator=g) * 0.05).to(dt)
    a = (torch.randn(r, K, generator=g) / K ** 0.5).to(dt)
    b = (torch.randn(N, r, generator=g) * 0.1).to(dt)
    return tuple(t.to(cuda) for t in (x, w, a, b))


def _dirty(cuda):
    """Leaves memory that the next buffers come from full of NaN bytes, so that a
    kernel which reads what nothing wrote, or too early, shows."""
    keep = [torch.full((n,), 255, dtype=torch.uint8, device=cuda)
            for n in (1 << 12, 1 << 16, 1 << 20, 1 << 24)]
    del keep


def _fwd_check(y, x, qw, a, b, alpha):
    dt, h = x.dtype, _half_step(x.dtype)
    r, K = a.shape
    s = alpha / r
    xq, _ = mx_oracle.mxfp4(_np(x))
    w = mx_oracle.unpack_fp4(qw.codes.cpu().numpy(), qw.scales.cpu().numpy())
    A, B, X = _np(a), _np(b), _np(x)
    xa = s * X @ A.T
    ref = xq @ w.T + xa @ B.T
    mag = np.abs(xq) @ np.abs(w).T + np.abs(xa) @ np.abs(B).T
    # s.x.A^T: an fp32 sum over K, then one rounding to 16 bits
    xa_err = K * ACC * (s * np.abs(X) @ np.abs(A).T) + h * np.abs(xa) + _tiny(dt)
    acc = xa_err @ np.abs(B).T + 1.01 * (K + r) * ACC * mag
    tol = acc + h * (np.abs(ref) + acc) + _tiny(dt)
    err = np.abs(_np(y) - ref)
    assert np.all(err <= tol), f"worst {np.max(err / np.maximum(tol, 1e-300))} of the bound"


SHAPES = [(1, 32, 8, 8), (1, 4096, 1024, 64), (2, 64, 24, 16), (16, 256, 128, 8), (15, 288, 136, 24),
          (17, 96, 1000, 16), (31, 160, 264, 8), (32, 512, 128, 32), (33, 544, 72, 16),
          (64, 1024, 384, 16), (65, 2080, 200, 128), (100, 128, 512, 256), (128, 320, 640, 16),
          (129, 256, 256, 16), (200, 4096, 264, 8), (256, 512, 256, 64), (257, 224, 520, 16),
          (300, 1056, 1000, 24), (513, 768, 768, 16), (16, 4096, 256, 16), (5, 928, 280, 16),
          (3, 3904, 136, 8), (30, 4224, 200, 64), (101, 5248, 136, 24), (59, 8160, 264, 32)]


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [BF16, FP16])
@pytest.mark.parametrize("M,K,N,r", SHAPES)
def test_forward(cuda, dt, M, K, N, r):
    x, w, a, b = _fwd_inputs(M, K, N, r, dt, cuda)
    qw = quant.quantize(w, "mxfp4")
    _dirty(cuda)
    y, saved = kernels.qlora_linear_fwd(x, qw, a, b, 32.0, save_xa=True)
    _fwd_check(y, x, qw, a, b, 32.0)
    _dirty(cuda)
    y2, none = kernels.qlora_linear_fwd(x, qw, a, b, 32.0)
    assert none is None and torch.equal(y, y2)  # bitwise repeatable
    with torch.no_grad():
        y3 = ops.qlora_forward(x, qw, a, b, 32.0)
    assert torch.equal(y, y3)
    # the rank intermediate the backward takes: (alpha/r) A.x^T, rows past r zero
    h = _half_step(dt)
    xa = 32.0 / r * _np(a) @ _np(x).T
    mag = 32.0 / r * np.abs(_np(a)) @ np.abs(_np(x)).T
    err = np.abs(_np(saved)[:r, :M] - xa)
    assert np.all(err <= (K * ACC * mag) * (1 + h) + h * np.abs(xa) + _tiny(dt))
    assert saved[r:, :M].abs().sum() == 0
    assert _lib.device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("M,K,N,r", [(4096, 4096, 136, 64), (2048, 4096, 264, 16), (16, 4096, 4096, 16),
                                     (1001, 4096, 2048, 64)])
def test_many_runs_agree(cuda, M, K, N, r):
    """A hundred passes back to back give the same bits, and the checkpoint the
    forward makes is the one of the pass of its own: a stage or a buffer handed
    on too early shows as a few wrong rows in one pass out of ten or so."""
    x, w, a, b = _fwd_inputs(M, K, N, r, BF16, cuda)
    dy = (torch.randn(M, N, generator=_gen(3)) * 0.1).to(BF16).to(cuda)
    qw = quant.quantize(w, "mxfp4")
    want = quant.checkpoint_activation(x)
    bad = torch.zeros(6, device=cuda)
    first = None
    for _ in range(100):
        c = quant.empty_checkpoint(x)
        y, saved = kernels.qlora_linear_fwd(x, qw, a, b, 32.0, save_xa=True, ckpt_out=c)
        _, da, db = kernels.lora_linear_bwd(dy, c, None, a, b, 32.0, saved, need_dx=False)
        got = (y, saved[:, :M], da, db)
        first = first or tuple(t.clone() for t in got)
        bad += torch.stack([(p != q).any().float() for p, q in zip(got, first)]
                           + [(c.codes != want.codes).any().float(),
                              (c.scales[:, :M] != want.scales[:, :M]).any().float()])
    assert bad.sum() == 0, bad.tolist()


@pytest.mark.gpu
def test_forward_nan_blocks(cuda):
    """A token with an infinity or a NaN gives a NaN row and touches no other;
    a NaN block of the weight gives a NaN output feature."""
    for M in (3, 40, 300):
        x, w, a, b = _fwd_inputs(M, 256, 264, 16, BF16, cuda)
        qw = quant.quantize(w, "mxfp4")
        y = kernels.qlora_linear_fwd(x, qw, a, b, 32.0)[0]
        x2 = x.clone()
        x2[1, 70] = float("inf")
        x2[2, 255] = float("nan")
        y2 = kernels.qlora_linear_fwd(x2, qw, a, b, 32.0)[0]
        keep = [i for i in range(M) if i not in (1, 2)]
        assert y2[1:3].isnan().all() and torch.equal(y2[keep], y[keep])
        w2 = w.clone()
        w2[5, 0] = float("-inf")
        y3 = kernels.qlora_linear_fwd(x, quant.quantize(w2, "mxfp4"), a, b, 32.0)[0]
        cols = [i for i in range(264) if i != 5]
        assert y3[:, 5].isnan().all() and torch.equal(y3[:, cols], y[:, cols])


@pytest.mark.gpu
def test_forward_c_abi_bounds(cuda):
    """The library builds the scale table when none is given, writes nothing past
    y, and refuses a workspace below the size it asks for."""
    lib = _lib.load()
    M, K, N, r = 130, 160, 136, 8
    x, w, a, b = _fwd_inputs(M, K, N, r, BF16, cuda)
    qw = quant.quantize(w, "mxfp4")
    want = kernels.qlora_linear_fwd(x, qw, a, b, 16.0)[0]
    y = torch.full((M + 8, N), 7.0, dtype=BF16, device=cuda)
    need = lib.mlora_qlora_forward_workspace_bytes(M, K, N, r, qw.code, 32)
    ws = torch.full((need + 256,), 255, dtype=torch.uint8, device=cuda)

    def call(nbytes):
        return lib.mlora_qlora_forward_ex(x.data_ptr(), qw.code, qw.codes.data_ptr(),
                                          qw.scales.data_ptr(), None, None, 32, a.data_ptr(),
                                          b.data_ptr(), y.data_ptr(), None, M, K, N, r, 16.0, 0,
                                          ws.data_ptr(), nbytes, kernels._stream())
    assert call(need - 256) == _lib.MLORA_ERR_WORKSPACE
    assert call(need) == 0
    assert torch.equal(y[:M], want) and (y[M:] == 7).all() and (ws[need:] == 255).all()


# ----------------------------------------------------------------- gradients --

def _ckpt_values(c):
    by = _mx_quant_scales(c).astype(np.float64)
    s = np.where(by == 255, np.nan, np.exp2(by - 127))
    return c.codes.cpu().numpy() / 64.0 * np.repeat(s, 32, -1)[:, : c.shape[-1]]


def _grad_check(da, db, dy, xh, saved, a, b, alpha, old=None, clip=None, parts=2):
    """dA = s (dy.B)^T.x^ with s dy.B in `parts` 16-bit parts, dB = dy^T.saved."""
    dt, h = dy.dtype, _half_step(dy.dtype)
    r, N, M = a.shape[0], b.shape[0], dy.shape[0]
    s = alpha / r
    DY, B, S = _np(dy), _np(b), _np(saved)[:r, :M]
    u = s * DY @ B
    u_err = N * ACC * (s * np.abs(DY) @ np.abs(B)) + h ** parts * np.abs(u) + _tiny(dt)
    ref_a, mag_a = u.T @ xh, np.abs(u).T @ np.abs(xh)
    # x^ itself is exact in bf16 and, above fp16's subnormals, in fp16
    x_err = 0.0 if dt == BF16 else np.abs(u).sum(0)[:, None] * _tiny(dt)
    tol_a = u_err.T @ np.abs(xh) + 1.01 * parts * M * ACC * mag_a + x_err
    ref_b, tol_b = DY.T @ S.T, M * ACC * (np.abs(DY).T @ np.abs(S).T)
    for got, ref, tol, o in ((da, ref_a, tol_a, 0), (db, ref_b, tol_b, 1)):
        if clip:
            ref = np.clip(ref, -clip, clip)
        if old is not None:
            ref = ref + _np(old[o])
        # the stored type's rounding (an accumulated sum rounds once more)
        g = 2 * ACC if got.dtype == FP32 else _half_step(got.dtype) + ACC
        tol = tol + g * (np.abs(ref) + tol) + (_tiny(got.dtype) if got.dtype != FP32 else 1e-40)
        err = np.abs(_np(got) - ref)
        assert np.all(err <= tol), f"worst {np.max(err / tol)} of the bound"


def _grad_inputs(M, K, N, r, dt, cuda, seed=0):
    x, w, a, b = _fwd_inputs(M, K, N, r, dt, cuda, seed)
    dy = (torch.randn(M, N, generator=_gen(seed + 3)) * 0.1).to(dt).to(cuda)
    _, saved = kernels.lora_linear_fwd(x, w, a, b, 32.0, save_xa=True)
    return x, w, a, b, dy, saved


GRAD_SHAPES = [(1, 8, 8, 8), (7, 40, 24, 16), (63, 128, 72, 8), (64, 64, 64, 16), (65, 200, 136, 24),
               (130, 264, 128, 32), (257, 1000, 264, 64), (300, 384, 200, 128), (515, 136, 64, 256),
               (1001, 512, 384, 16), (2048, 256, 128, 8), (4099, 128, 64, 64)]


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [BF16, FP16])
@pytest.mark.parametrize("M,K,N,r", GRAD_SHAPES)
def test_gradients_from_checkpoint(cuda, dt, M, K, N, r):
    x, w, a, b, dy, saved = _grad_inputs(M, K, N, r, dt, cuda)
    _dirty(cuda)
    c = quant.checkpoint_activation(x)
    xh = _ckpt_values(c)
    for gdt in (None, dt):
        _dirty(cuda)
        dx, da, db = kernels.lora_linear_bwd(dy, c, None, a, b, 32.0, saved, need_dx=False,
                                             grad_dtype=gdt)
        assert dx is None and da.dtype == db.dtype == (gdt or FP32)
        _grad_check(da, db, dy, xh, saved, a, b, 32.0)
    da2, db2 = ops.lora_backward(dy, c, a, b, 32.0, clip_value=None, saved_xa=saved)
    assert torch.equal(da, da2) and torch.equal(db, db2)  # bitwise repeatable
    da3, db3 = ops.lora_backward(dy, c, a, b, 32.0, clip_value=0.05, saved_xa=saved)
    _grad_check(da3, db3, dy, xh, saved, a, b, 32.0, clip=0.05)
    # added into fp32 buffers
    old = (torch.randn(r, K, generator=_gen(5)).to(cuda), torch.randn(N, r, generator=_gen(6)).to(cuda))
    acc = tuple(t.clone() for t in old)
    kernels.lora_linear_bwd(dy, c, None, a, b, 32.0, saved, need_dx=False, da_out=acc[0],
                            db_out=acc[1], accumulate=True)
    _grad_check(*acc, dy, xh, saved, a, b, 32.0, old=old)
    # without the saved intermediate dB comes from the checkpoint's values too
    xq = c.dequantize()
    da4, db4 = ops.lora_backward(dy, c, a, b, 32.0, clip_value=None)
    da5, db5 = ops.lora_backward(dy, xq, a, b, 32.0, clip_value=None)
    assert torch.equal(da4, da5) and torch.equal(db4, db5)
    assert _lib.device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [BF16, FP16])
def test_gradient_extreme_scales(cuda, dt):
    """Blocks at both ends of the exponent range (the bf16 top end takes the
    kernel's multiplying form), zero blocks, and a NaN block."""
    M, K, N, r = 70, 128, 64, 8
    x, w, a, b, dy, saved = _grad_inputs(M, K, N, r, dt, cuda)
    x = torch.randn(M, K, generator=_gen(9)).to(cuda)
    top, low = (120.0, -126.0) if dt == BF16 else (14.0, -14.0)
    x[:, 0:32] *= 2.0 ** top / 8
    x[:, 32:64] *= 2.0 ** low
    x[:, 64:96] = 0
    c = quant.checkpoint_activation(x.to(dt))
    dy[:, :] = torch.randint(-1, 2, dy.shape, device=cuda).to(dt) * 2.0 ** -6
    _, da, db = kernels.lora_linear_bwd(dy, c, None, a, b, 8.0, saved, need_dx=False)
    assert torch.isfinite(da).all() and (da[:, 64:96] == 0).all()
    _grad_check(da, db, dy, _ckpt_values(c), saved, a, b, 8.0)
    x[3, 100] = float("nan")
    c = quant.checkpoint_activation(x.to(dt))
    _, da2, db2 = kernels.lora_linear_bwd(dy, c, None, a, b, 8.0, saved, need_dx=False)
    assert da2[:, 96:].isnan().all() and torch.equal(da2[:, :96], da[:, :96])
    assert torch.equal(db2, db)


@pytest.mark.gpu
def test_gradient_c_abi_bounds(cuda):
    """Rows of codes between K and the row stride are not read, nothing is
    written past dA."""
    M, K, N, r = 77, 200, 64, 8
    x, w, a, b, dy, saved = _grad_inputs(M, K, N, r, BF16, cuda)
    c = quant.checkpoint_activation(x)
    wide = torch.full((M, 256), 99, dtype=torch.int8, device=cuda)
    wide[:, :K] = c.codes
    c2 = quant.ActivationCheckpoint(wide[:, :K], c.scales, c.shape, c.dtype)
    buf = torch.full((r * K + 64,), 5.0, device=cuda)
    db = torch.empty(N, r, device=cuda)
    da = buf[: r * K].view(r, K)
    kernels.lora_linear_bwd(dy, c2, None, a, b, 32.0, saved, need_dx=False, da_out=da, db_out=db,
                            accumulate=False)
    _, want, _ = kernels.lora_linear_bwd(dy, c, None, a, b, 32.0, saved, need_dx=False)
    assert torch.equal(da, want) and (buf[r * K:] == 5).all()


@pytest.mark.gpu
def test_gradient_refusals(cuda):
    x, w, a, b, dy, saved = _grad_inputs(16, 64, 64, 8, BF16, cuda)
    c = quant.checkpoint_activation(x)
    def call(c=c, saved=saved, dy=dy):
        return kernels.lora_linear_bwd(dy, c, None, a, b, 32.0, saved, need_dx=False)
    call()
    with pytest.raises(ShapeError):  # needs the forward's intermediate
        call(saved=None)
    with pytest.raises(ShapeError):
        call(saved=saved[:8])
    with pytest.raises(ShapeError):
        call(dy=dy.half())
    with pytest.raises(ShapeError):
        call(c=quant.checkpoint_activation(x.float()))
    with pytest.raises(ShapeError):
        call(c=quant.checkpoint_activation(x[:8]))
    qw = quant.quantize(w, "mxfp4")
    with pytest.raises(ShapeError):
        kernels.qlora_linear_fwd(x.float(), qw, a.float(), b.float(), 32.0)
    with pytest.raises(ShapeError):
        ops.qlora_forward(x, qw, a.requires_grad_(), b, 32.0, checkpoint=quant.checkpoint_activation(x[:8]))
    w48 = quant.quantize(torch.randn(64, 48, device=cuda, dtype=BF16), "mxfp4")
    with pytest.raises(ShapeError):  # the product wants whole blocks
        kernels.qlora_linear_fwd(x[:, :48], w48, a[:, :48].detach(), b, 32.0)


# -------------------------------------------------------------- used together --

def _step(x, qw, a, b, dy, checkpoint):
    leaves = [t.detach().clone().requires_grad_(True) for t in (x, a, b)]
    y = ops.qlora_forward(leaves[0], qw, leaves[1], leaves[2], 32.0, checkpoint=checkpoint)
    return y.detach(), *torch.autograd.grad(y, leaves, dy)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [BF16, FP16])
@pytest.mark.parametrize("M,K,N,r", [(5, 64, 24, 8), (100, 288, 136, 20), (300, 512, 264, 64),
                                     (20, 4096, 72, 16)])
def test_step(cuda, dt, M, K, N, r):
    """Forward and backward over an MXFP4 base with and without a checkpoint:
    the checkpoint changes dA alone; dx = dy.W + s (dy.B).A."""
    x, w, a, b = _fwd_inputs(M, K, N, r, dt, cuda)
    dy = (torch.randn(M, N, generator=_gen(4)) * 0.1).to(dt).to(cuda)
    qw = quant.quantize(w, "mxfp4")
    _dirty(cuda)
    y, dx, da, db = _step(x, qw, a, b, dy, "mxint8")
    _dirty(cuda)
    y0, dx0, da0, db0 = _step(x, qw, a, b, dy, None)
    shared = quant.checkpoint_activation(x)
    y1, dx1, da1, db1 = _step(x, qw, a, b, dy, shared)
    assert torch.equal(y, y0) and torch.equal(dx, dx0) and torch.equal(db, db0)
    assert all(torch.equal(p, q) for p, q in ((y, y1), (dx, dx1), (da, da1), (db, db1)))
    _fwd_check(y, x, qw, a, b, 32.0)
    _, saved = kernels.qlora_linear_fwd(x, qw, a, b, 32.0, save_xa=True)
    _grad_check(da, db, dy, _ckpt_values(shared), saved, a, b, 32.0)
    _grad_check(da0, db0, dy, _np(x), saved, a, b, 32.0, parts=1)
    h, s = _half_step(dt), 32.0 / r
    W = mx_oracle.unpack_fp4(qw.codes.cpu().numpy(), qw.scales.cpu().numpy())
    DY, A, B = _np(dy), _np(a), _np(b)
    u = s * DY @ B
    ref = DY @ W + u @ A
    mag = np.abs(DY) @ np.abs(W) + np.abs(u) @ np.abs(A)
    u_err = N * ACC * (s * np.abs(DY) @ np.abs(B)) + h * np.abs(u) + _tiny(dt)
    # W is exact in bf16 and above fp16's subnormals in fp16
    w_err = 0.0 if dt == BF16 else np.abs(DY).sum(1, keepdims=True) * _tiny(dt)
    acc = u_err @ np.abs(A) + 1.01 * (N + r) * ACC * mag + w_err
    assert np.all(np.abs(_np(dx) - ref) <= acc + h * (np.abs(ref) + acc) + _tiny(dt))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [BF16, FP16])
@pytest.mark.parametrize("K", [8, 40, 200, 232, 1000, 1056, 4096])
def test_forward_writes_the_checkpoint(cuda, dt, K):
    """The checkpoint a forward makes is the one of ``checkpoint_activation``, at
    every value the format has to round, saturate or refuse, word padding
    included; the forward's own outputs are those without it."""
    e = _edge_rows(dt)
    x = torch.cat([e.repeat(1, -(-K // e.shape[1]))[:, :K],
                   e.flip(1).repeat(1, -(-K // e.shape[1]))[:, :K], _acts(151, K, dt, 2)]).to(cuda)
    g = _gen(1)
    w = (torch.randn(72, K, generator=g) * 0.05).to(dt).to(cuda)
    a = (torch.randn(16, K, generator=g) / K ** 0.5).to(dt).to(cuda)
    b = (torch.randn(72, 16, generator=g) * 0.1).to(dt).to(cuda)
    want = quant.checkpoint_activation(x)
    runs = [lambda o: kernels.lora_linear_fwd(x, w, a, b, 32.0, save_xa=True, ckpt_out=o)]
    if K % 32 == 0:
        qw = quant.quantize(w, "mxfp4")
        runs.append(lambda o: kernels.qlora_linear_fwd(x, qw, a, b, 32.0, save_xa=True, ckpt_out=o))
    for run in runs:
        _dirty(cuda)
        got = quant.empty_checkpoint(x)
        y, saved = run(got)
        assert torch.equal(got.codes, want.codes)
        assert torch.equal(got.scales[:, : x.shape[0]], want.scales[:, : x.shape[0]])
        y0, saved0 = run(None)
        same = ~(torch.isnan(y) & torch.isnan(y0))
        assert torch.equal(y[same], y0[same])
        M = x.shape[0]
        same = ~(torch.isnan(saved[:, :M]) & torch.isnan(saved0[:, :M]))
        assert torch.equal(saved[:, :M][same], saved0[:, :M][same])


@pytest.mark.gpu
def test_gradients_against_differences(cuda):
    """On inputs whose roundings are exact (a grid both formats hold) the
    forward is linear in A and B, so central differences of the kernel's own
    forward give <dy, y'> = <dA, A'> and <dB, B'> up to y's rounding."""
    M, K, N, r, dt = 96, 128, 64, 8, BF16
    g = _gen(11)
    pick = torch.tensor([-1.0, -0.5, 0.0, 0.5, 1.0, 1.5])
    x = pick[torch.randint(0, 6, (M, K), generator=g)].to(dt).to(cuda)
    w = (torch.randn(N, K, generator=g) * 0.05).to(dt).to(cuda)
    a = (torch.randint(-4, 5, (r, K), generator=g) / 64).to(dt).to(cuda)
    b = (torch.randint(-4, 5, (N, r), generator=g) / 64).to(dt).to(cuda)
    dy = (torch.randint(-8, 9, (M, N), generator=g) / 16).to(dt).to(cuda)
    qw = quant.quantize(w, "mxfp4")
    c = quant.checkpoint_activation(x)
    assert torch.equal(c.dequantize(), x) and torch.equal(quant.quantize(x, "mxfp4").dequantize(dt), x)
    _, dx, da, db = _step(x, qw, a, b, dy, c)
    h = _half_step(dt)

    def fwd(a_, b_):
        return _np(kernels.qlora_linear_fwd(x, qw, a_, b_, 8.0)[0])
    DY = _np(dy)
    for which, grad in (("a", da), ("b", db)):
        p = a if which == "a" else b
        step = (torch.randint(-1, 2, p.shape, generator=g) / 16).to(dt).to(cuda)
        hi = fwd(p + step, b) if which == "a" else fwd(a, p + step)
        lo = fwd(p - step, b) if which == "a" else fwd(a, p - step)
        diff = (DY * (hi - lo)).sum() / 2
        want = (_np(grad) * _np(step)).sum()
        # y's and s.x.A^T's roundings in both forwards, the gradient's own
        y_err = h * (np.abs(hi) + np.abs(lo)) / 2
        X, A, B, P = (np.abs(_np(t)) for t in (x, a, b, step))
        xa = X @ (A + (P if which == "a" else 0)).T      # s = 1
        xa_err = h * xa @ (B + (P if which == "b" else 0)).T
        tol = (np.abs(DY) * (1.01 * y_err + xa_err)).sum() + 1.01 * h * np.abs(_np(grad) * _np(step)).sum()
        if which == "a":  # dA's rounded s dy.B
            tol += ((h * np.abs(DY) @ B).T @ X * P).sum()
        else:             # dB's rounded s x.A^T
            tol += (np.abs(DY).T @ (h * xa) * P).sum()
        assert abs(diff - want) <= tol, (which, diff, want, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("scheme", [None, "nf4", "int4", "mxfp4"])
def test_layers_share_a_checkpoint(cuda, scheme):
    """Three projections of one input keep one checkpoint; every base takes it."""
    torch.manual_seed(0)
    layers = [LoRALinear(256, n, rank=16, alpha=32.0, device=cuda, dtype=BF16) for n in (256, 64, 72)]
    for m in layers:
        with torch.no_grad():
            m.W0.normal_(0, 0.05)
            m.B.normal_(0, 0.05)
        if scheme:
            m.quantize_base(scheme)
    x = _acts(96, 256, BF16, 3).to(cuda).view(4, 24, 256).requires_grad_(True)
    c = quant.checkpoint_activation(x)

    def grads(ckpt):
        out = [m(x, checkpoint=ckpt) for m in layers]
        loss = sum((o.float() ** 2).sum() for o in out)
        return torch.autograd.grad(loss, [x] + [t for m in layers for t in (m.A, m.B)])
    shared = grads(c)
    for m in layers:
        m.activation_checkpoint = "mxint8"
    own = grads(None)
    assert all(torch.equal(p, q) for p, q in zip(shared, own))
    for m in layers:
        m.activation_checkpoint = None
    plain = grads(None)
    # dx and dB are those of the 16-bit x; dA differs by the checkpoint's rounding
    for i, (p, q) in enumerate(zip(shared, plain)):
        if i == 0 or i % 2 == 0:
            assert torch.equal(p, q), i


@pytest.mark.gpu
def test_checkpoint_saves_memory(cuda):
    """What the backward holds of x is the 8-bit form, not x."""
    m = LoRALinear(2048, 64, rank=8, device=cuda, dtype=BF16, activation_checkpoint="mxint8")
    saved = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: saved.append(t) or t, lambda t: t):
        x = torch.randn(512, 2048, device=cuda, dtype=BF16)
        m(x)
    assert not any(t.dtype == BF16 and t.shape == x.shape for t in saved)
    held = [t for t in saved if t.dtype in (torch.int8, torch.uint8)]
    assert sum(t.numel() for t in held) == 512 * 2048 * 33 // 32


@pytest.mark.gpu
def test_trainer_with_checkpoints(cuda, tmp_path):
    """The trainer's flat buffers, accumulation and split backward take the
    checkpoint's gradients: one step equals the layers' own gradients."""
    def model():
        torch.manual_seed(1)
        net = torch.nn.Sequential(LoRALinear(128, 192, rank=8, device=cuda, dtype=BF16),
                                  LoRALinear(192, 64, rank=8, device=cuda, dtype=BF16))
        with torch.no_grad():
            for m in net:
                m.W0.normal_(0, 0.1)
                m.B.normal_(0, 0.1)
        return net.apply(lambda m: m.quantize_base("mxfp4") if isinstance(m, LoRALinear) else None)
    x = _acts(64, 128, BF16, 5).to(cuda).view(2, 32, 128)
    t = torch.randn(2, 32, 64, device=cuda)
    tr = LoRATrainer(model(), TrainingConfig(activation_checkpoint="mxint8", max_grad_norm=0.0,
                                             gradient_accumulation_steps=2, output_dir=str(tmp_path)))
    assert all(m.activation_checkpoint == "mxint8" for m in tr.model)
    tr.backward({"input_ids": x, "target_output": t})
    tr.backward({"input_ids": x, "target_output": t})
    net = model()
    for m in net:
        m.activation_checkpoint = "mxint8"
    loss = torch.mean((net(x).float() - t) ** 2)
    for (name, m), ref in zip(tr.params.layers, net):
        ga, gb = torch.autograd.grad(loss, (ref.A, ref.B), retain_graph=True)
        oa, na, sa = tr.params.slices[f"{name}.A"]
        ob, nb, sb = tr.params.slices[f"{name}.B"]
        # the trainer's fp32 sums against the same sums rounded to bf16
        for got, want in ((tr.params.grad[oa:oa + na].view(sa), ga), (tr.params.grad[ob:ob + nb].view(sb), gb)):
            # (two exact halves of one gradient add up exactly)
            want = _np(want)
            h = _half_step(BF16)
            assert np.all(np.abs(_np(got) - want) <= h * np.abs(want) * (1 + 2 * h) + _tiny(BF16))
    tr.optimizer_step()
    assert torch.isfinite(tr.params.master).all()


@pytest.mark.gpu
def test_custom_operator_takes_mxfp4(cuda):
    from metallora_b200 import torch_ops
    x, w, a, b = _fwd_inputs(48, 256, 136, 16, BF16, cuda)
    dy = torch.randn(48, 136, generator=_gen(8)).to(BF16).to(cuda)
    qw = quant.quantize(w, "mxfp4")
    y, dx, da, db = _step(x, qw, a, b, dy, None)
    leaves = [t.detach().clone().requires_grad_(True) for t in (x, a, b)]
    y2 = torch_ops.qlora_linear(leaves[0], qw, leaves[1], leaves[2], 32.0)
    got = torch.autograd.grad(y2, leaves, dy)
    assert torch.equal(y, y2) and all(torch.equal(p, q) for p, q in zip((dx, da, db), got))


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 40, 300])
def test_streams_and_graphs(cuda, M):
    """Two streams at once and two captured graphs give the eager results."""
    x, w, a, b = _fwd_inputs(M, 512, 264, 16, BF16, cuda)
    dy = torch.randn(M, 264, generator=_gen(8)).to(BF16).to(cuda)
    qw = quant.quantize(w, "mxfp4")
    x2 = x.flip(0).contiguous()
    want = [_step(v, qw, a, b, dy, "mxint8") for v in (x, x2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [None, None]
    for _ in range(3):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i] = _step((x, x2)[i], qw, a, b, dy, "mxint8")
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(p, q) for p, q in zip(got[i], want[i]))
    # forward and checkpoint backward captured (kernel calls: no autograd graph)
    def run(v, y, da):
        out, saved = kernels.qlora_linear_fwd(v, qw, a, b, 32.0, save_xa=True)
        c = quant.checkpoint_activation(v)
        _, g, _ = kernels.qlora_linear_bwd(dy, c, qw, a, b, 32.0, saved, need_dx=True)
        y.copy_(out)
        da.copy_(g)
    graphs, outs, static = [], [], [x.clone(), x2.clone()]
    for v in static:
        y, da = torch.empty(M, 264, dtype=BF16, device=cuda), torch.empty(16, 512, device=cuda)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            run(v, y, da)
        graphs.append(graph)
        outs.append((y, da))
    for _ in range(2):
        for graph in graphs:
            graph.replay()
    torch.cuda.synchronize()
    for i, (y, da) in enumerate(outs):
        assert torch.equal(y, want[i][0])
        assert torch.equal(da.to(BF16), want[i][2])
    static[0].copy_(x2)
    graphs[0].replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0][0], want[1][0]) and torch.equal(outs[0][1].to(BF16), want[1][2])


@pytest.mark.gpu
def test_first_use_inside_a_capture(cuda):
    """A weight that is first multiplied while a graph is captured is right
    eagerly before the graph has ever run, and in the graph."""
    x, w, a, b = _fwd_inputs(20, 256, 136, 16, BF16, cuda)
    want = kernels.qlora_linear_fwd(x, quant.quantize(w, "mxfp4"), a, b, 32.0)[0]
    q0 = quant.quantize(w, "mxfp4")
    fresh = quant.QuantizedWeight("mxfp4", q0.codes, q0.scales, None, 32, q0.shape)  # no table yet
    y = torch.zeros_like(want)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y.copy_(kernels.qlora_linear_fwd(x, fresh, a, b, 32.0)[0])
    _dirty(cuda)
    assert torch.equal(kernels.qlora_linear_fwd(x, fresh, a, b, 32.0)[0], want)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, want)


@pytest.mark.gpu
def test_empty_batch(cuda):
    x, w, a, b = _fwd_inputs(4, 64, 24, 8, BF16, cuda)
    qw = quant.quantize(w, "mxfp4")
    y, dx, da, db = _step(x[:0], qw, a, b, torch.empty(0, 24, dtype=BF16, device=cuda), "mxint8")
    assert y.shape == (0, 24) and dx.shape == (0, 64) and not da.any() and not db.any()


# ------------------------------------------------- calls at the edges of the API --

def test_weight_parts_refusals():
    """The kernels size their reads by the shape: parts that do not fit it, or a
    table of another size, are refused however the weight was made."""
    codes, scales = torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 2, dtype=torch.uint8)
    ok = dict(scheme="mxfp4", codes=codes, scales=scales, zeros=None, group=32, shape=(4, 64))
    qw = quant.QuantizedWeight(**ok)
    for change in ({"codes": codes[:3]}, {"scales": scales[:, :1]}, {"scales": scales.float()},
                   {"codes": codes.t().contiguous().t()}, {"zeros": scales}, {"group": 64},
                   {"lean": True}, {"shape": (4, 66)},
                   {"shape": (4, 65), "scales": torch.zeros(4, 3, dtype=torch.uint8)},
                   {"scales": scales.to("meta")}):
        with pytest.raises(QuantizationError):
            quant.QuantizedWeight(**{**ok, **change})
    qw.check_table(torch.zeros(512, dtype=torch.uint8))
    for bad in (torch.zeros(511, dtype=torch.uint8), torch.zeros(512, dtype=torch.int8),
                torch.zeros(1024, dtype=torch.uint8)[::2],
                torch.zeros(512, dtype=torch.uint8, device="meta")):
        with pytest.raises(ShapeError):
            qw.check_table(bad)


def test_gradient_buffer_refusals():
    """Host tensors and wrong shapes are refused before any launch."""
    saved = torch.zeros(16, 8, dtype=BF16)
    with pytest.raises(DeviceError):
        kernels._check_saved(saved, 8, 7, BF16)
    for bad in (saved[:8], saved.half()):
        with pytest.raises(ShapeError):
            kernels._check_saved(bad, 8, 7, BF16)
    da, db = torch.zeros(8, 64), torch.zeros(24, 8)
    with pytest.raises(DeviceError):
        kernels._check_grad_out(da, db, 8, 8, 64, 24)
    for bad in ((None, db, 8, 8), (da, None, 8, 8), (da.half(), db, 8, 8), (da[:, :32], db, 8, 8),
                (da, db.t().contiguous().t(), 8, 8), (da, db, 8, 7)):
        with pytest.raises(ShapeError):
            kernels._check_grad_out(*bad, 64, 24)


def test_too_many_tokens_are_refused():
    """Past 2^31 - 256 tokens a row number of the last tile would not fit 32 bits."""
    lib = _lib.load()
    buf = C.create_string_buffer(1 << 12)
    p = (C.addressof(buf) + 255) // 256 * 256
    mx = _lib.QUANT_MXFP4
    for M in ((1 << 31) - 255, (1 << 31) - 1, 1 << 31):
        rc = lib.mlora_qlora_forward_ex(p, mx, p, p, None, p, 32, p, p, p, None, M, 32, 8, 8, 1.0, 0, p,
                                        1 << 10, None)
        assert rc == _lib.MLORA_ERR_UNSUPPORTED, M


@pytest.mark.gpu
def test_more_refusals(cuda):
    x, w, a, b, dy, saved = _grad_inputs(16, 64, 64, 8, BF16, cuda)
    qw, c = quant.quantize(w, "mxfp4"), quant.checkpoint_activation(x)
    with pytest.raises(ShapeError):  # a weight of other sizes than dy and x
        kernels.qlora_linear_bwd(dy, x, quant.quantize(w[:32], "mxfp4"), a, b, 32.0, saved)
    with pytest.raises(DeviceError):
        ops.lora_backward(dy, c, a, b, 32.0, saved_xa=saved.cpu())
    for bad in ("fp8", quant.checkpoint_activation(x[:8])):
        with torch.no_grad(), pytest.raises(MetalLoRAError):
            ops.qlora_forward(x, qw, a, b, 32.0, checkpoint=bad)
    table = qw.prepared_scales()
    with pytest.raises(ShapeError):
        torch.ops.metal_lora.qlora_fwd(x, qw.codes, qw.scales, None, table[:256], "mxfp4", 32, False, a,
                                       b, 32.0)


@pytest.mark.gpu
@pytest.mark.parametrize("K", [1000, 1024])
def test_checkpoint_through_saved_tensor_hooks(cuda, K):
    """Offloaded to the host between forward and backward (which closes the gaps
    between the rows of K 1000), a checkpoint gives the same gradients."""
    x, w, a, b = _fwd_inputs(70, K, 72, 16, BF16, cuda)
    dy = torch.randn(70, 72, generator=_gen(8)).to(BF16).to(cuda)
    leaves = [t.requires_grad_(True) for t in (x, a, b)]
    want = torch.autograd.grad(ops.lora_forward(x, w, a, b, 32.0, checkpoint="mxint8"), leaves, dy)
    with torch.autograd.graph.save_on_cpu():
        y = ops.lora_forward(x, w, a, b, 32.0, checkpoint="mxint8")
    got = torch.autograd.grad(y, leaves, dy)
    assert all(torch.equal(p, q) for p, q in zip(want, got))


@pytest.mark.gpu
def test_loaded_bases_bring_their_table(cuda, tmp_path):
    """A loaded MXFP4 base has its table before its first product, whichever
    stream that runs on."""
    from metallora_b200.utils import load_quantized_bases, save_quantized_bases

    def net():
        torch.manual_seed(3)
        m = torch.nn.Sequential(LoRALinear(96, 136, rank=8, device=cuda, dtype=BF16))
        with torch.no_grad():
            m[0].W0.normal_(0, 0.1)
            m[0].B.normal_(0, 0.1)
        return m
    m = net()
    m[0].quantize_base("mxfp4")
    save_quantized_bases(m, tmp_path)
    m2 = load_quantized_bases(net(), tmp_path)
    assert getattr(m2[0].qweight, "_prepared", None) is not None
    x = _acts(33, 96, BF16, 1).to(cuda)
    assert torch.equal(m(x), m2(x))


@pytest.mark.gpu
def test_host_threads(cuda):
    """Two host threads, each on its stream, get the serial results."""
    import threading
    x, w, a, b = _fwd_inputs(200, 512, 264, 16, BF16, cuda)
    dy = torch.randn(200, 264, generator=_gen(8)).to(BF16).to(cuda)
    qw = quant.quantize(w, "mxfp4")
    inputs = [(x, dy), (x.flip(0).contiguous(), dy.flip(0).contiguous())]
    want = [_step(v, qw, a, b, d, "mxint8") for v, d in inputs]
    torch.cuda.synchronize()
    got, failed = [None, None], []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    got[i] = _step(inputs[i][0], qw, a, b, inputs[i][1], "mxint8")
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # noqa: BLE001
            failed.append(e)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(120)
    assert not failed, failed
    for i in range(2):
        assert all(torch.equal(p, q) for p, q in zip(got[i], want[i]))


@pytest.mark.gpu
def test_thread_without_a_context(cuda):
    """The first CUDA work of a host thread may be any of the calls: its buffers
    come from the allocator's cache, so nothing before has bound a context."""
    import threading
    x, w, a, b, dy, saved = _grad_inputs(70, 1024, 72, 16, BF16, cuda)
    qw, c = quant.quantize(w, "mxfp4"), quant.checkpoint_activation(x)
    calls = [lambda: kernels.lora_linear_fwd(x, w, a, b, 32.0, save_xa=True),
             lambda: kernels.qlora_linear_fwd(x, qw, a, b, 32.0, save_xa=True),
             lambda: kernels.lora_linear_bwd(dy, c, w, a, b, 32.0, saved),
             lambda: kernels.qlora_linear_bwd(dy, c, qw, a, b, 32.0, saved),
             lambda: (quant.checkpoint_activation(x).dequantize(), qw.dequantize(BF16))]
    for call in calls:
        want, got = call(), []

        def work():
            try:
                got.append(call())
            except Exception as e:  # noqa: BLE001
                got.append(e)
        t = threading.Thread(target=work)
        t.start()
        t.join(60)
        assert got and not isinstance(got[0], Exception), got
        torch.cuda.synchronize()
        # (rows past the tokens of saved_xa are not written)
        assert all(torch.equal(p[:, :70], q[:, :70]) for p, q in zip(want, got[0]))


@pytest.mark.gpu
def test_captured_training_step(cuda):
    """Forward and backward through autograd captured once, replayed on new inputs."""
    x, w, a, b = _fwd_inputs(150, 288, 136, 16, BF16, cuda)
    dy = torch.randn(150, 136, generator=_gen(8)).to(BF16).to(cuda)
    qw = quant.quantize(w, "mxfp4")
    want = [_step(v, qw, a, b, dy, "mxint8") for v in (x, x.flip(0).contiguous())]
    leaves = [t.detach().clone().requires_grad_(True) for t in (x, a, b)]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = ops.qlora_forward(leaves[0], qw, leaves[1], leaves[2], 32.0, checkpoint="mxint8")
        grads = torch.autograd.grad(y, leaves, dy)
    for v, ref in ((x, want[0]), (x.flip(0), want[1]), (x, want[0])):
        with torch.no_grad():
            leaves[0].copy_(v)
        _dirty(cuda)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p.detach(), q) for p, q in zip((y, *grads), ref))


@pytest.mark.gpu
def test_split_backward_of_a_checkpoint(cuda):
    """The two-call backward gives the one call's results, added and written."""
    x, w, a, b, dy, saved = _grad_inputs(150, 288, 136, 16, BF16, cuda)
    c = quant.checkpoint_activation(x)
    dx, da, db = kernels.lora_linear_bwd(dy, c, w, a, b, 32.0, saved)
    for accumulate in (False, True):
        ga, gb = torch.ones_like(da), torch.ones_like(db)
        finish = kernels.lora_linear_bwd_split(dy, c, w, a, b, 32.0, saved, ga, gb, accumulate=accumulate)
        _dirty(cuda)
        assert torch.equal(finish(), dx)
        assert torch.equal(ga, da + 1 if accumulate else da)
        assert torch.equal(gb, db + 1 if accumulate else db)


@pytest.mark.gpu
def test_offsets_past_32_bits(cuda):
    """More than 2^31 elements in x, y and dy: the last rows are those of the same
    call on them alone, and gradients of a dy that is zero elsewhere theirs."""
    M, K, N, r, n = 264200, 8192, 8200, 16, 200
    g = torch.Generator(device=cuda).manual_seed(0)
    x = torch.randn(M, K, device=cuda, dtype=BF16, generator=g)
    w = torch.randn(N, K, device=cuda, dtype=BF16, generator=g) * 0.05
    a = torch.randn(r, K, device=cuda, dtype=BF16, generator=g) / K ** 0.5
    b = torch.randn(N, r, device=cuda, dtype=BF16, generator=g) * 0.1
    qw = quant.quantize(w, "mxfp4")
    tail = x[-n:].clone()
    c = quant.checkpoint_activation(x)
    ct = quant.checkpoint_activation(tail)
    assert torch.equal(c.codes[-n:], ct.codes) and torch.equal(c.scales[:, M - n:M], ct.scales[:, :n])
    assert torch.equal(c.dequantize()[-n:], ct.dequantize())
    made = quant.empty_checkpoint(x)
    y, saved = kernels.qlora_linear_fwd(x, qw, a, b, 32.0, save_xa=True, ckpt_out=made)
    assert torch.equal(made.codes, c.codes) and torch.equal(made.scales[:, :M], c.scales[:, :M])
    del c
    _fwd_check(y[-16:], tail[-16:], qw, a, b, 32.0)
    del y, x
    dy = torch.zeros(M, N, device=cuda, dtype=BF16)
    dy[-n:] = torch.randn(n, N, device=cuda, dtype=BF16, generator=g) * 0.1
    _, da, db = kernels.lora_linear_bwd(dy, made, None, a, b, 32.0, saved, need_dx=False)
    # (adding exact zeros changes no partial sum: the bound of the n rows holds)
    _grad_check(da, db, dy[-n:], _ckpt_values(ct), saved[:, M - n:M], a, b, 32.0)
    assert _lib.device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("M,K,N", [(1, 4096, 1024), (64, 1024, 1024), (700, 1024, 512)])
def test_calls_that_follow_their_producers(cuda, M, K, N):
    """Every call may start while the kernel before it still runs: one that reads
    what the call just before it wrote gives the results of waiting in between."""
    x, w, a, b = _fwd_inputs(M, K, N, 16, BF16, cuda)
    dy = torch.randn(M, N, generator=_gen(8)).to(BF16).to(cuda)

    def chain(wait):
        def then(v):
            if wait:
                torch.cuda.synchronize()
            return v
        ck = then(quant.checkpoint_activation(then(x * 1)))
        back = then(ck.dequantize())
        qw = then(quant.quantize(then(w + 0), "mxfp4"))
        y, saved = then(kernels.qlora_linear_fwd(back, qw, a, b, 32.0, save_xa=True))
        made = quant.empty_checkpoint(back)
        y2, _ = then(kernels.qlora_linear_fwd(back, qw, a, b, 32.0, save_xa=True, ckpt_out=made))
        grads = then(kernels.qlora_linear_bwd(then(y2 * dy), made, qw, a, b, 32.0, saved))
        again = then(kernels.lora_linear_bwd(then(dy * 1), then(quant.checkpoint_activation(back)),
                                             then(qw.dequantize(BF16)), a, b, 32.0, saved))
        return (ck.codes, back, y, y2, made.codes, *grads, *again)
    want = chain(True)
    for _ in range(20):
        _dirty(cuda)
        assert all(torch.equal(p, q) for p, q in zip(chain(False), want))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [BF16, FP16])
@pytest.mark.parametrize("M,K,N,r", [(1290, 128, 2048, 16), (2600, 96, 2104, 24), (2570, 320, 4000, 8)])
def test_forward_waves(cuda, dt, M, K, N, r):
    """More tiles than half a wave (whole ones), whole ones and halves in one call."""
    x, w, a, b = _fwd_inputs(M, K, N, r, dt, cuda)
    qw = quant.quantize(w, "mxfp4")
    _dirty(cuda)
    y, _ = kernels.qlora_linear_fwd(x, qw, a, b, 32.0)
    _fwd_check(y, x, qw, a, b, 32.0)
    assert torch.equal(y[:200], kernels.qlora_linear_fwd(x[:200], qw, a, b, 32.0)[0])
    assert _lib.device_status() == 0


@pytest.mark.gpu
def test_capture_with_joined_streams(cuda):
    """Captured calls that come first, follow a copy or a fill, or follow a join of
    two streams (their producer is on the other one) replay as they run."""
    x, w, a, b = _fwd_inputs(70, 256, 136, 16, BF16, cuda)
    dy = torch.randn(70, 136, generator=_gen(8)).to(BF16).to(cuda)
    qw = quant.quantize(w, "mxfp4")
    xs, side = x.clone(), torch.cuda.Stream()
    buf, scratch = torch.empty_like(x), torch.empty(1 << 20, dtype=torch.uint8, device=cuda)

    def run():
        outs = [quant.checkpoint_activation(xs).codes]
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            buf.copy_(xs * 2)
        scratch.zero_()
        torch.cuda.current_stream().wait_stream(side)
        y, saved = kernels.qlora_linear_fwd(buf, qw, a, b, 32.0, save_xa=True)
        scratch.fill_(1)
        c = quant.checkpoint_activation(buf)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            back = c.dequantize()
            g = dy * 3
        scratch.zero_()
        torch.cuda.current_stream().wait_stream(side)
        outs += [y, back, *kernels.qlora_linear_bwd(g, c, qw, a, b, 32.0, saved)]
        return outs
    want = [t.clone() for t in run()]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run()
    for _ in range(3):
        _dirty(cuda)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(got, want))
    xs.copy_(x.flip(0))
    want = [t.clone() for t in run()]
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(got, want))
