"""Calls over MXFP4 bases and MXINT8 checkpoints that the formats' own tests leave
out: derivatives that the operators do not define, values that are not finite, parts
changed in place, every base with a checkpoint, products that are exact.
"""
import copy
import ctypes
import pickle

import pytest
import torch
from torch.autograd import forward_ad

from metallora_b200 import _lib, kernels, ops, quant, trainer
from metallora_b200.exceptions import AdapterError, ConfigurationError
from metallora_b200.layers import LoRALinear
from metallora_b200.trainer import LoRATrainer, TrainingConfig

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _cpu_weight(n=24, k=64):
    return quant.from_reference_layout("mxfp4", torch.zeros((n, k // 2), dtype=torch.uint8),
                                       torch.full((n, k // 32), 127, dtype=torch.uint8), None, (n, k), 32)


def _inputs(M, K, N, r, dt, cuda, seed=0):
    g = _gen(seed + M + K + N)
    x = torch.randn(M, K, generator=g)
    w = torch.randn(N, K, generator=g) * 0.05
    a = torch.randn(r, K, generator=g) / K ** 0.5
    b = torch.randn(N, r, generator=g) * 0.1
    dy = torch.randn(M, N, generator=g) * 0.1
    return tuple(t.to(dt).to(cuda) for t in (x, w, a, b, dy))


# ----------------------------------------------------------------- derivatives --

@pytest.mark.parametrize("which", ["x", "a", "b"])
def test_forward_mode_is_refused(monkeypatch, which):
    """The operator has no forward-mode rule: a dual tensor is refused, with
    gradients switched off too, and never answered without its tangent."""
    qw = _cpu_weight()
    monkeypatch.setattr(kernels, "qlora_linear_fwd",
                        lambda x, q, a, b, alpha, save_xa=False, ckpt_out=None: (
                            x.new_zeros((x.shape[0], q.shape[0])),
                            x.new_zeros((16, (x.shape[0] + 7) // 8 * 8)) if save_xa else None))
    t = {"x": torch.randn(6, 64, dtype=BF16), "a": torch.randn(8, 64, dtype=BF16),
         "b": torch.randn(24, 8, dtype=BF16)}
    assert ops.qlora_forward(t["x"], qw, t["a"], t["b"]).shape == (6, 24)
    with forward_ad.dual_level():
        dual = {**t, which: forward_ad.make_dual(t[which], torch.ones_like(t[which]))}
        with pytest.raises(NotImplementedError):
            ops.qlora_forward(dual["x"], qw, dual["a"], dual["b"])
        with torch.no_grad(), pytest.raises(NotImplementedError):
            ops.qlora_forward(dual["x"], qw, dual["a"], dual["b"])
        assert ops.qlora_forward(t["x"], qw, t["a"], t["b"]).shape == (6, 24)


# ------------------------------------------------------- values that are not finite --

@pytest.mark.gpu
@pytest.mark.parametrize("dt", [BF16, FP16])
@pytest.mark.parametrize("r", [8, 64, 128])
def test_clip_keeps_nan(cuda, dt, r):
    """Clipping bounds numbers: a gradient that is NaN stays NaN, with the default
    clip, from a checkpoint and from x itself, whatever the gradients' type."""
    M, K, N = 150, 256, 72
    x, w, a, b, dy = _inputs(M, K, N, r, dt, cuda)
    x[3, 70] = float("nan")   # block 2 of row 3
    x[9, 250] = float("inf")  # block 7 of row 9
    _, saved = kernels.lora_linear_fwd(torch.nan_to_num(x, 0.0, 1.0), w, a, b, 32.0, save_xa=True)
    c = quant.checkpoint_activation(x)
    dead = torch.zeros(K, dtype=torch.bool, device=cuda)
    dead[64:96] = dead[224:256] = True
    dirty = dy.clone()
    dirty[5, 11] = float("nan")
    for gdt in (None, dt):
        _, da0, db0 = kernels.lora_linear_bwd(dy, c, None, a, b, 32.0, saved, need_dx=False,
                                              grad_dtype=gdt)
        _, da, db = kernels.lora_linear_bwd(dy, c, None, a, b, 32.0, saved, clip_value=0.0625,
                                            need_dx=False, grad_dtype=gdt)
        assert da[:, dead].isnan().all() and torch.equal(db, db0.clamp(-0.0625, 0.0625))
        assert torch.equal(da[:, ~dead], da0[:, ~dead].clamp(-0.0625, 0.0625))
        _, da, db = kernels.lora_linear_bwd(dirty, c, None, a, b, 32.0, saved, clip_value=0.0625,
                                            need_dx=False, grad_dtype=gdt)
        assert db[11].isnan().all() and not torch.cat([db[:11], db[12:]]).isnan().any()
        assert da.isnan().all()
    da, db = ops.lora_backward(dirty, c, a, b, 32.0, saved_xa=saved)  # clips at 1
    assert da.isnan().all() and db[11].isnan().all()
    # from x itself
    da, db = ops.lora_backward(dy, x, a, b, 32.0, saved_xa=saved)
    cols = torch.zeros(K, dtype=torch.bool, device=cuda)
    cols[70] = True
    assert da[:, cols].isnan().all() and not da[:, ~cols & ~dead].isnan().any()
    da, db = ops.lora_backward(dirty, x, a, b, 32.0, saved_xa=saved)
    assert da.isnan().all() and db[11].isnan().all()


@pytest.mark.gpu
def test_clip_keeps_nan_fp32(cuda):
    x, w, a, b, dy = _inputs(40, 64, 72, 8, FP32, cuda)
    dy[5, 11] = float("nan")
    da, db = ops.lora_backward(dy, x, a, b, 16.0)
    assert da.isnan().all() and db[11].isnan().all()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [BF16, FP16])
@pytest.mark.parametrize("r", [8, 64])
def test_infinite_intermediate(cuda, dt, r):
    """An infinite s dy B, made by an infinite dy or by passing fp16's largest number,
    is an infinity with its sign in dA as well."""
    M, K, N = 70, 128, 64
    x, w, a, b, dy = _inputs(M, K, N, r, dt, cuda)
    x = x.abs() + 0.5
    dy.zero_()
    dy[4] = 100.0 if dt == FP16 else float("inf")
    b[:, 0], b[:, 1] = 50.0, -50.0  # 4 * 64 * 100 * 50 is 20 times fp16's largest
    b[:, 2:] = 0.25                 # 4 * 64 * 100 / 4 is a tenth of it
    _, saved = kernels.lora_linear_fwd(x, w, a, b, 4.0 * r, save_xa=True)
    c = quant.checkpoint_activation(x)
    for clip, big in ((0.0, float("inf")), (1.0, 1.0)):
        _, da, _ = kernels.lora_linear_bwd(dy, c, None, a, b, 4.0 * r, saved, clip_value=clip,
                                           need_dx=False)
        assert (da[0] == big).all() and (da[1] == -big).all()
        assert torch.isfinite(da[2:]).all() if dt == FP16 else (da[2:] == big).all()


# ------------------------------------------------------------------ the scale table --

@pytest.mark.gpu
@pytest.mark.parametrize("scheme", ["mxfp4", "nf4", "int4", "int8"])
def test_parts_changed_in_place(cuda, scheme):
    """A weight whose scales are written over multiplies by the new ones."""
    dt = BF16
    x, w, a, b, dy = _inputs(4, 256, 72, 8, dt, cuda)
    qw = quant.quantize(w, scheme)
    other = quant.quantize(w * 4, scheme)
    kernels.qlora_linear_fwd(x, qw, a, b, 16.0)
    for part in ("codes", "scales", "zeros"):
        if getattr(qw, part) is not None:
            getattr(qw, part).copy_(getattr(other, part))
    for M in (1, 4):
        want = kernels.qlora_linear_fwd(x[:M], quant.quantize(w * 4, scheme), a, b, 16.0)[0]
        assert torch.equal(kernels.qlora_linear_fwd(x[:M], qw, a, b, 16.0)[0], want)
    with torch.inference_mode():
        q2 = quant.quantize(w, scheme)
        y = kernels.qlora_linear_fwd(x, q2, a, b, 16.0)[0]
    for _ in range(2):  # (and out of it)
        assert torch.equal(y, kernels.qlora_linear_fwd(x, q2, a, b, 16.0)[0])
    # a copy has scales of its own
    twin, y = copy.deepcopy(qw), kernels.qlora_linear_fwd(x, qw, a, b, 16.0)[0]
    assert torch.equal(kernels.qlora_linear_fwd(x, twin, a, b, 16.0)[0], y)
    for part in ("codes", "scales", "zeros"):
        if getattr(qw, part) is not None:
            getattr(twin, part).copy_(getattr(q2, part))
    assert torch.equal(kernels.qlora_linear_fwd(x, twin, a, b, 16.0)[0],
                       kernels.qlora_linear_fwd(x, q2, a, b, 16.0)[0])
    assert torch.equal(kernels.qlora_linear_fwd(x, qw, a, b, 16.0)[0], y)
    # other tensors in the place of the parts
    qw.codes, qw.scales, qw.zeros = twin.codes, twin.scales, twin.zeros
    assert torch.equal(kernels.qlora_linear_fwd(x, qw, a, b, 16.0)[0],
                       kernels.qlora_linear_fwd(x, q2, a, b, 16.0)[0])


@pytest.mark.gpu
@pytest.mark.parametrize("scheme", ["mxfp4", "int4"])
def test_graphs_follow_a_changed_weight(cuda, scheme):
    """A graph captured before a weight's parts were written over replays with the new
    weight once its table has been made anew: it never reads a table that is gone."""
    x, w, a, b, _ = _inputs(4, 256, 72, 8, BF16, cuda)
    qw, other = quant.quantize(w, scheme), quant.quantize(w.flip(0) * 4, scheme)
    kernels.qlora_linear_fwd(x, qw, a, b, 16.0)
    y = torch.empty(4, 72, dtype=BF16, device=cuda)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y.copy_(kernels.qlora_linear_fwd(x, qw, a, b, 16.0)[0])
    for part in ("codes", "scales", "zeros"):
        if getattr(qw, part) is not None:
            getattr(qw, part).copy_(getattr(other, part))
    want = kernels.qlora_linear_fwd(x, other, a, b, 16.0)[0]
    assert torch.equal(kernels.qlora_linear_fwd(x, qw, a, b, 16.0)[0], want)
    keep = [torch.full((n,), 255, dtype=torch.uint8, device=cuda) for n in (512, 1 << 12, 1 << 16, 1 << 20)]
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, want) and len(keep) == 4


def test_copies_of_a_weight():
    """A copied or pickled weight holds its parts and no table of another's."""
    qw = _cpu_weight()
    qw._keep_table(torch.zeros(512, dtype=torch.uint8))
    assert qw._kept_table() is qw._prepared
    for twin in (copy.deepcopy(qw), copy.copy(qw), pickle.loads(pickle.dumps(qw))):
        assert twin.shape == qw.shape and twin.scheme == "mxfp4" and twin._kept_table() is None
        assert torch.equal(twin.codes, qw.codes) and torch.equal(twin.scales, qw.scales)
    qw.scales.add_(1)
    assert qw._kept_table() is None
    qw._keep_table(torch.zeros(512, dtype=torch.uint8))
    qw.scales = qw.scales.clone()
    assert qw._kept_table() is None


def _files(tmp_path, shapes):
    weights = {name: _cpu_weight(n, k) for name, (n, k) in shapes.items()}
    quant.save_quantized(weights, tmp_path / "base.safetensors")


# ----------------------------------------------------------------------- settings --

def test_table_of_another_device(monkeypatch):
    """A weight that is loaded onto a GPU which is not the current one gets its table
    there, in that device's context."""
    events = []

    class Guard:
        def __init__(self, device):
            self.device = device

        def __enter__(self):
            events.append(("in", self.device))

        def __exit__(self, *exc):
            events.append(("out", self.device))

    class Weight:
        scheme = "mxfp4"

        class codes:
            is_cuda, device = True, torch.device("cuda:1")

            @staticmethod
            def get_device():
                return 1

        scales = codes

        def prepared_scales(self):
            events.append("table")
    monkeypatch.setattr(torch.cuda, "device", Guard)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    quant._with_table(Weight())
    assert events == [("in", torch.device("cuda:1")), "table", ("out", torch.device("cuda:1"))]


def test_loading_is_all_or_nothing(tmp_path):
    """A file that does not fit the model leaves every module as it was."""
    from metallora_b200.utils import load_quantized_bases

    def net():
        return torch.nn.Sequential(LoRALinear(64, 24, rank=8), LoRALinear(64, 40, rank=8))
    for second in ((48, 64), (40, 96)):
        _files(tmp_path, {"0": (24, 64), "1": second})
        m = net()
        with pytest.raises(AdapterError):
            load_quantized_bases(m, tmp_path)
        assert all(l.qweight is None and l.W0.numel() for l in m)
    _files(tmp_path, {"0": (24, 64), "other": (40, 64)})
    m = net()
    with pytest.raises(AdapterError):
        load_quantized_bases(m, tmp_path)
    assert all(l.qweight is None and l.W0.numel() for l in m)
    _files(tmp_path, {"0": (24, 64), "1": (40, 64)})
    m = load_quantized_bases(net(), tmp_path)
    assert all(l.qweight is not None and not l.W0.numel() for l in m)


def test_checkpoint_settings_are_checked_first(tmp_path):
    """What the layers' forward would refuse, the trainer refuses before it touches
    the model; what it would take is taken."""
    def config(**kw):
        return TrainingConfig(activation_checkpoint="mxint8", rank=8, output_dir=str(tmp_path), **kw)

    def lora(dtype=BF16, **kw):
        return torch.nn.Sequential(LoRALinear(64, 64, rank=8, dtype=dtype, **kw))

    def plain(dtype):
        return torch.nn.ModuleDict({"q_proj": torch.nn.Linear(64, 64, dtype=dtype),
                                    "head": torch.nn.Linear(64, 64)})
    for model, kw in ((lora(dropout=0.1), {}), (lora(FP32), {}), (plain(BF16), {"dropout": 0.1}),
                      (plain(FP32), {})):
        before = [(n, type(m)) for n, m in model.named_modules()]
        grads = [p.requires_grad for p in model.parameters()]
        with pytest.raises(ConfigurationError):
            LoRATrainer(model, config(**kw))
        assert [(n, type(m)) for n, m in model.named_modules()] == before
        assert [p.requires_grad for p in model.parameters()] == grads
        assert not any(getattr(m, "activation_checkpoint", None) for m in model.modules())
    off = lora(dropout=0.1).eval()  # dropout that is switched off is none
    quantised = lora(FP32, dropout=0.1)
    quantised[0].qweight = _cpu_weight(64, 64)
    trainer._check_activation_checkpoint(plain(BF16), config())
    trainer._check_activation_checkpoint(off, config())
    trainer._check_activation_checkpoint(quantised, config())
    trainer._check_activation_checkpoint(plain(FP32), TrainingConfig(dropout=0.1))


def test_c_abi_wants_whole_elements():
    """An address inside an element would fault in the kernel: it is refused."""
    lib = _lib.load()
    buf = ctypes.create_string_buffer(1 << 12)
    p = (ctypes.addressof(buf) + 255) // 256 * 256
    mx, bad = _lib.QUANT_MXFP4, _lib.MLORA_ERR_INVALID_ARG
    for dtype, off in ((0, 1), (1, 1), (2, 2)):
        assert lib.mlora_quantize(p + off, dtype, 4, 64, mx, 32, p, p, None, None) == bad
        assert lib.mlora_quantize(p + off, dtype, 4, 64, _lib.QUANT_NF4, 64, p, p, None, None) == bad
        assert lib.mlora_quantize_mxfp4(p + off, dtype, 4, 64, p, p, p, None) == bad
        assert lib.mlora_dequantize(mx, p, p, None, 4, 64, 32, p + off, dtype, None) == bad
        assert lib.mlora_act_checkpoint(p + off, dtype, 4, 64, p, 64, p, None) == bad
        assert lib.mlora_act_restore(p, 64, p, 4, 64, p + off, dtype, None) == bad
        assert b"whole element" in lib.mlora_last_error_message()


@pytest.mark.parametrize("M", [(1 << 31) - 255, (1 << 31) - 1, 1 << 31])
def test_checkpoints_of_too_many_tokens_are_refused(M):
    """Past 2^31 - 256 tokens a row number of the last tile would not fit 32 bits."""
    K, N = 64, 64
    lib = _lib.load()
    buf = ctypes.create_string_buffer(1 << 12)
    p = (ctypes.addressof(buf) + 255) // 256 * 256
    mx, no = _lib.QUANT_MXFP4, _lib.MLORA_ERR_UNSUPPORTED
    sizes, ld = (M, K, N, 8, 1.0), K
    assert lib.mlora_lora_forward_ckpt(p, p, p, p, p, p, p, ld, p, *sizes, 0, p, 1 << 10, None) == no
    assert lib.mlora_lora_backward_ckpt(p, p, ld, p, None, p, p, p, None, p, p, *sizes, 0.0, 0, 0, p,
                                        1 << 10, None) == no
    assert lib.mlora_qlora_forward_ckpt(p, mx, p, p, None, p, 32, p, p, p, p, p, ld, p, *sizes, 0, p,
                                        1 << 10, None) == no
    assert lib.mlora_qlora_backward_ckpt(p, p, ld, p, mx, p, p, None, p, 32, p, p, p, p, p, p, *sizes,
                                         0.0, 0, 0, p, 1 << 10, None) == no


# ---------------------------------------------------------- every base, exact products --

@pytest.mark.gpu
@pytest.mark.parametrize("dt", [BF16, FP16])
@pytest.mark.parametrize("M,K,N,r", [(1, 4096, 264, 64), (16, 4096, 1024, 16), (40, 4096, 136, 8),
                                     (100, 8160, 136, 24), (128, 4096, 264, 128), (300, 4096, 520, 16),
                                     (700, 4096, 264, 64), (1290, 4128, 2048, 16)])
def test_exact_products(cuda, dt, M, K, N, r):
    """Operands that the formats hold, with sums that fp32 holds at every step: y
    is the 64-bit result rounded once, bit for bit.  |x|, |w| <= 1.5 in halves, one
    power of two a token and one (1, 2) a block of w: a term is a multiple of 1/4, a
    sum at most 4.5 K < 2^18 quarters.  A has 8 entries +-1 a row, so that x A^T is a
    multiple of 1/2 up to 12 (24 halves: 5 bits); B holds multiples of 1/4 up to 1, and
    the rank term adds at most 12 r, in eighths."""
    g = _gen(M + K + N + r)
    pick = torch.tensor([-1.5, -1.0, -0.5, 0.0, 0.5, 1.0, 1.5])
    x = pick[torch.randint(0, 7, (M, K), generator=g)]
    x *= torch.exp2(torch.randint(-2, 3, (M, 1), generator=g).float())
    w = pick[torch.randint(0, 7, (N, K), generator=g)]
    w *= torch.exp2(torch.randint(0, 2, (N, K // 32), generator=g).float()).repeat_interleave(32, 1)
    a = torch.zeros(r, K)
    for j in range(r):
        at = torch.randperm(K, generator=g)[:8]
        a[j, at] = torch.randint(0, 2, (8,), generator=g).float() * 2 - 1
    b = torch.randint(-4, 5, (N, r), generator=g) / 4
    ref = x.double() @ w.double().t() + (x.double() @ a.double().t()) @ b.double().t()
    x, w, a, b = (t.to(dt).to(cuda) for t in (x, w, a, b.float()))
    qw = quant.quantize(w, "mxfp4")
    assert torch.equal(qw.dequantize(dt), w) and torch.equal(quant.quantize(x, "mxfp4").dequantize(dt), x)
    y = kernels.qlora_linear_fwd(x, qw, a, b, float(r))[0]
    assert torch.equal(y.cpu(), ref.float().to(dt))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [BF16, FP16])
@pytest.mark.parametrize("M", [3, 40, 300])
@pytest.mark.parametrize("r", [8, 16, 24, 64, 128, 200])
def test_rank_term_is_rounded_once(cuda, dt, M, r):
    """s x A^T goes to its product with B unrounded: with x A^T of 13 significant bits
    (multiples of 1/16 up to 384; the 16-bit types hold 8 and 11), y is still the 64-bit
    result rounded once.  The sums stay below 2^24 steps of 1/64."""
    K, N = 256, 136
    g = _gen(M + r)
    pick = torch.tensor([-1.5, -1.0, -0.5, 0.0, 0.5, 1.0, 1.5])
    x, w = pick[torch.randint(0, 7, (M, K), generator=g)], pick[torch.randint(0, 7, (N, K), generator=g)]
    a = torch.randint(-8, 9, (r, K), generator=g) / 8
    b = torch.randint(-4, 5, (N, r), generator=g) / 4
    xa = x.double() @ a.double().t()
    assert (xa != xa.to(BF16).double()).any()
    ref = x.double() @ w.double().t() + xa @ b.double().t()
    x, w, a, b = (t.to(dt).to(cuda) for t in (x, w, a, b))
    y, saved = kernels.qlora_linear_fwd(x, quant.quantize(w, "mxfp4"), a, b, float(r), save_xa=True)
    assert torch.equal(y.cpu(), ref.float().to(dt))
    assert torch.equal(saved[:r, :M].cpu(), xa.t().float().to(dt))  # (kept rounded)


@pytest.mark.gpu
@pytest.mark.parametrize("lean", [False, True])
@pytest.mark.parametrize("scheme", ["nf4", "int4", "int8"])
@pytest.mark.parametrize("M", [1, 16, 90, 300])
def test_checkpoint_over_quantised_bases(cuda, scheme, lean, M):
    """Over every base, lean weights included, a checkpoint leaves y and dx as they
    are without it, is the one of ``checkpoint_activation``, and gives dA of its values."""
    K, N, r = 256, 136, 16
    x, w, a, b, dy = _inputs(M, K, N, r, BF16, cuda)
    qw = quant.quantize(w, scheme, lean=lean)
    made = quant.empty_checkpoint(x)
    y0, saved0 = kernels.qlora_linear_fwd(x, qw, a, b, 32.0, save_xa=True)
    y, saved = kernels.qlora_linear_fwd(x, qw, a, b, 32.0, save_xa=True, ckpt_out=made)
    want = quant.checkpoint_activation(x)
    assert torch.equal(made.codes, want.codes) and torch.equal(made.scales[:, :M], want.scales[:, :M])
    assert torch.equal(y, y0) and torch.equal(saved[:, :M], saved0[:, :M])
    y1, none = kernels.qlora_linear_fwd(x, qw, a, b, 32.0, ckpt_out=made)  # nothing saved
    assert none is None and torch.equal(made.codes, want.codes) and torch.equal(y1, y0)
    dx0, _, db0 = kernels.qlora_linear_bwd(dy, x, qw, a, b, 32.0, saved)
    dx, da, db = kernels.qlora_linear_bwd(dy, made, qw, a, b, 32.0, saved)
    dx2, da2, db2 = kernels.lora_linear_bwd(dy, made, None, a, b, 32.0, saved, need_dx=False)
    assert dx2 is None and torch.equal(da, da2) and torch.equal(db, db2)
    for x_ in (x, made):  # 16-bit gradients are the fp32 ones rounded
        _, wa, wb = kernels.qlora_linear_bwd(dy, x_, qw, a, b, 32.0, saved)
        _, ha, hb = kernels.qlora_linear_bwd(dy, x_, qw, a, b, 32.0, saved, grad_dtype=BF16)
        assert torch.equal(ha, wa.to(BF16)) and torch.equal(hb, wb.to(BF16))
    half = torch.finfo(BF16).eps / 2
    u = 2.0 * dy.double() @ b.double()
    acc = N * 2.0 ** -23 * 2.0 * dy.double().abs() @ b.double().abs()  # fp32 sums of U
    # U's 16-bit rounding in dx, twice where the two differ; the fp32 sums of both
    # products; the two results' own roundings
    mag = dy.double().abs() @ qw.dequantize(FP32).double().abs() + u.abs() @ a.double().abs()
    tol = 2 * ((half * u.abs() + acc) @ a.double().abs() + (N + r) * 2.0 ** -22 * mag)
    tol = tol + half * (dx.double().abs() + dx0.double().abs()) * (1 + half)
    assert ((dx.double() - dx0.double()).abs() <= tol).all()
    ref = u.t() @ made.dequantize(FP32).double()
    tol = (half ** 2 * u.abs() + acc).t() @ made.dequantize(FP32).double().abs() + \
        2.02 * M * 2.0 ** -23 * u.abs().t() @ made.dequantize(FP32).double().abs() + 2.0 ** -22 * ref.abs()
    assert ((da.double() - ref).abs() <= tol + 1e-40).all()
    S = saved[:r, :M].double()
    tol = (M + 2) * 2.0 ** -23 * dy.double().abs().t() @ S.abs().t()
    assert ((db.double() - dy.double().t() @ S.t()).abs() <= tol + 1e-40).all()
    assert ((db.double() - db0.double()).abs() <= 2 * tol + 1e-40).all()
    assert _lib.device_status() == 0
