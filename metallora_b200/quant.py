"""Quantised base weights (NF4, group-wise INT4/INT8) for QLoRA.

Storage follows the reference shaders' layout (kernels/lora_quantized.metal):
packed codes ``[N, K/2]`` bytes with the low nibble holding the even k
(:70-74) -- ``[N, K]`` for INT8 -- and per-row, per-block scales:
fp32 absmax ``[N, ceil(K/group)]`` for NF4 (:122, :135), fp16 scale and zero
``[N, ceil(K/group)]`` for INT4/INT8 (the reference's per-row int4 is
``group = K``).  ``quantize`` runs on the GPU (the reference ships no
quantiser); ``dequantize`` returns fp32 values bit-identical to the
reference's ``dequant_nf4``/``dequant_int4``.

Two formats have no reference counterpart.  Both give 32 consecutive features
of a row one power-of-two factor ``2^E``, kept as the byte ``E + 127``:

* MXFP4 weights (``quantize(w, "mxfp4")``): ``w = e2m1 * 2^E`` with ``E =
  floor(log2 max|w|) - 2``, codes packed as NF4's, scales uint8
  ``[N, ceil(K/32)]``.  The forward multiplies them by activations rounded to
  the same format, on the fp4 tensor cores, with nothing dequantised.
* MXINT8 activation checkpoints (``checkpoint_activation(x)``): ``x = code / 64
  * 2^E`` with ``E = floor(log2 max|x|)``.  The LoRA backward takes one in the
  place of x, at half the bytes of a 16-bit x.

E is at least -127; a block that holds an infinity or a NaN reads back as NaN.
"""
from __future__ import annotations

from dataclasses import dataclass

import torch

from . import _lib
from .exceptions import DeviceError, QuantizationError, ShapeError
from .kernels import _dtype_code, _need_cuda, _need_current, _ptr, _stream

SCHEMES = {"nf4": _lib.QUANT_NF4, "int4": _lib.QUANT_INT4, "int8": _lib.QUANT_INT8,
           "mxfp4": _lib.QUANT_MXFP4}
DEFAULT_GROUP = {"nf4": 64, "int4": 128, "int8": 128, "mxfp4": 32}
_SCALE_DTYPE = {"nf4": torch.float32, "int4": torch.float16, "int8": torch.float16,
                "mxfp4": torch.uint8}
_WITH_ZEROS = ("int4", "int8")


@dataclass
class QuantizedWeight:
    """A quantised [out_features, in_features] weight."""
    scheme: str
    codes: torch.Tensor
    scales: torch.Tensor
    zeros: torch.Tensor | None
    group: int
    shape: tuple[int, int]
    lean: bool = False  # fused in-loop dequant (no transient bf16 copy of W per call)

    def __post_init__(self):
        if self.scheme == "mxfp4":
            self._check_mxfp4_parts()

    def _check_mxfp4_parts(self) -> None:
        """The kernels size their reads by ``shape`` alone, so the parts have to fit it."""
        _check_mxfp4(self.scheme, self.group, self.lean)
        N, K = self.shape
        for part, t, shp in (("codes", self.codes, (N, K // 2)),
                             ("scales", self.scales, (N, -(-K // 32)))):
            if t.dtype != torch.uint8 or tuple(t.shape) != shp or not t.is_contiguous():
                raise QuantizationError(f"mxfp4 {part}: expected contiguous {shp} uint8, got "
                                        f"{tuple(t.shape)} {t.dtype}")
        if K % 2:
            raise QuantizationError("4-bit codes pack two per byte: in_features must be even")
        if self.codes.device != self.scales.device:
            raise QuantizationError("mxfp4 codes and scales are on different devices")
        if self.zeros is not None:
            raise QuantizationError("mxfp4 has no zero points")

    @property
    def code(self) -> int:
        return SCHEMES[self.scheme]

    @property
    def device(self):
        return self.codes.device

    def nbytes(self) -> int:
        n = self.codes.numel() + self.scales.numel() * self.scales.element_size()
        if self.zeros is not None:
            n += self.zeros.numel() * self.zeros.element_size()
        return n

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        return dequantize(self, dtype)

    def _kept_table(self) -> torch.Tensor | None:
        """The kept scale table, if it is of these scales and zeros as they are now."""
        kept = getattr(self, "_table_of", None)
        if kept is None or self._prepared.device != self.codes.device:
            return None
        s, z = self.scales, self.zeros
        # (what is written over through .data or in inference mode keeps no count of it)
        if kept[0] is s and kept[1] is z and kept[2] == (-1 if s.is_inference() else s._version) and \
                (z is None or kept[3] == (-1 if z.is_inference() else z._version)):
            return self._prepared
        return None

    def _keep_table(self, table: torch.Tensor) -> None:
        s, z = self.scales, self.zeros
        self._prepared = table
        self._table_of = (s, z, -1 if s.is_inference() else s._version,
                          -1 if z is None or z.is_inference() else z._version)

    def __getstate__(self):
        """A copy's tensors count their writes anew: it makes its own table."""
        return {k: v for k, v in self.__dict__.items() if k not in ("_prepared", "_table_of")}

    def __setstate__(self, state) -> None:
        self.__dict__.update(state)
        _with_table(self)

    def prepared_scales(self) -> torch.Tensor:
        """The TMA-ready scale table the GPU kernels read: [groups, rows rounded
        to 4], or for MXFP4 the product's blocks of 128 rows x 128 features
        (built on first use -- for MXFP4 when the weight is made -- and kept with
        the weight; a table built while a graph is captured belongs to that graph and
        is not kept).  Once the scales or zeros are written over it is made anew, in
        the same memory: graphs captured with it replay with the new one."""
        t = self._kept_table()
        if t is None:
            lib = _lib.load()
            N, K = self.shape
            capturing = torch.cuda.is_current_stream_capturing()
            kept = getattr(self, "_table_of", None)
            if kept is not None and kept[0] is self.scales and kept[1] is self.zeros and \
                    self._prepared.device == self.codes.device and not capturing:
                t = self._prepared
            else:
                nbytes = lib.mlora_qlora_prepared_scales_bytes(self.code, N, K, self.group)
                t = torch.empty(nbytes, dtype=torch.uint8, device=self.codes.device)
            st = lib.mlora_qlora_prepare_scales(self.code, _ptr(self.scales), _ptr(self.zeros), N,
                                                K, self.group, _ptr(t), _stream())
            _lib.check(st, "mlora_qlora_prepare_scales")
            if not capturing:
                self._keep_table(t)
        return t

    def check_table(self, table: torch.Tensor) -> None:
        """Raises unless ``table`` has the size of this weight's ``prepared_scales``."""
        N, K = self.shape
        need = _lib.load().mlora_qlora_prepared_scales_bytes(self.code, N, K, self.group)
        if table.dtype != torch.uint8 or table.numel() != need or not table.is_contiguous() or \
                table.device != self.codes.device:
            raise ShapeError(f"the prepared scales must be {need} contiguous bytes on "
                             f"{self.codes.device}, got {tuple(table.shape)} {table.dtype} on "
                             f"{table.device}")

    def state_dict(self) -> dict[str, torch.Tensor]:
        d = {"codes": self.codes, "scales": self.scales}
        if self.zeros is not None:
            d["zeros"] = self.zeros
        return d


def _check_mxfp4(scheme: str, group, lean: bool) -> None:
    if scheme != "mxfp4":
        return
    if group not in (None, 0, 32):
        raise QuantizationError(f"mxfp4 blocks hold 32 features, got group {group}")
    if lean:
        raise QuantizationError("mxfp4 has no lean form: its forward dequantises nothing")


def quantize(w: torch.Tensor, scheme: str = "nf4", group: int | None = None,
             lean: bool = False) -> QuantizedWeight:
    """Quantises a 2-D CUDA weight [N, K] (bf16/fp16/fp32).  ``lean`` makes the
    LoRA kernels dequantise inside the GEMM main loop instead of staging a
    bf16 copy of the weight in their workspace (less memory, slower); MXFP4,
    whose forward stages nothing, takes neither it nor another group."""
    if scheme not in SCHEMES:
        raise QuantizationError(f"unknown scheme {scheme!r}; use one of {sorted(SCHEMES)}")
    _check_mxfp4(scheme, group, lean)
    _need_cuda(w)
    if w.dim() != 2:
        raise ShapeError("quantize takes a 2-D weight [out_features, in_features]")
    group = group or DEFAULT_GROUP[scheme]
    N, K = w.shape
    if scheme == "mxfp4":
        return _quantize_mxfp4(w.contiguous())
    if scheme != "int8" and K % 2:
        raise QuantizationError("4-bit codes pack two per byte: in_features must be even")
    G = -(-K // group)
    w = w.contiguous()
    dev = w.device
    codes = torch.empty((N, K if scheme == "int8" else K // 2), dtype=torch.uint8, device=dev)
    scales = torch.empty((N, G), dtype=_SCALE_DTYPE[scheme], device=dev)
    zeros = torch.empty((N, G), dtype=torch.float16, device=dev) if scheme in _WITH_ZEROS else None
    st = _lib.load().mlora_quantize(_ptr(w), _dtype_code(w), N, K, SCHEMES[scheme], group,
                                    _ptr(codes), _ptr(scales), _ptr(zeros), _stream())
    _lib.check(st, "mlora_quantize")
    return QuantizedWeight(scheme, codes, scales, zeros, group, (N, K), lean)


def _quantize_mxfp4(w: torch.Tensor) -> QuantizedWeight:
    _need_current(w)
    N, K = w.shape
    if N == 0 or K == 0:
        raise ShapeError("quantize takes a weight with at least one row and one column")
    lib = _lib.load()
    codes = w.new_empty((N, K // 2), dtype=torch.uint8)
    scales = w.new_empty((N, -(-K // 32)), dtype=torch.uint8)
    table = w.new_empty(lib.mlora_qlora_prepared_scales_bytes(_lib.QUANT_MXFP4, N, K, 32),
                        dtype=torch.uint8)
    st = lib.mlora_quantize_mxfp4(w.data_ptr(), _dtype_code(w), N, K, codes.data_ptr(),
                                  scales.data_ptr(), table.data_ptr(), _stream())
    _lib.check(st, "mlora_quantize_mxfp4")
    qw = QuantizedWeight("mxfp4", codes, scales, None, 32, (N, K))
    qw._keep_table(table)
    return qw


def _with_table(qw: QuantizedWeight) -> QuantizedWeight:
    """An MXFP4 weight on the GPU gets its table at once, in the order of its codes
    on its device's stream: no later call, on whatever stream, is the one that makes
    it."""
    if qw.scheme == "mxfp4" and qw.codes.is_cuda:
        with torch.cuda.device(qw.codes.device):
            qw.prepared_scales()
    return qw


def dequantize(qw: QuantizedWeight, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """Dense [N, K] weights: fp32 = the reference's dequantised values (bit
    exact); bf16/fp16 = those values rounded, the operand the GEMMs use."""
    N, K = qw.shape
    if qw.scheme == "mxfp4":
        _need_current(qw.codes)
    out = qw.codes.new_empty((N, K), dtype=dtype)
    st = _lib.load().mlora_dequantize(qw.code, _ptr(qw.codes), _ptr(qw.scales), _ptr(qw.zeros), N,
                                      K, qw.group, _ptr(out), _dtype_code(out), _stream())
    _lib.check(st, "mlora_dequantize")
    return out


def from_reference_layout(scheme: str, codes, scales, zeros, shape, group,
                          lean: bool = False) -> QuantizedWeight:
    """Wraps tensors already in the reference layout (e.g. loaded from disk)."""
    if scheme not in SCHEMES:
        raise QuantizationError(f"unknown scheme {scheme!r}")
    return _with_table(QuantizedWeight(scheme, codes.contiguous(), scales.contiguous(),
                                       None if zeros is None else zeros.contiguous(), int(group),
                                       (int(shape[0]), int(shape[1])), lean))


# ------------------------------------------------- activation checkpoints --

@dataclass
class ActivationCheckpoint:
    """The MXINT8 form of activations x, kept for the backward instead of x.

    ``codes`` int8 [M, K], rows a multiple of 16 bytes apart; ``scales`` uint8
    [ceil(K/128), M rounded up to 4, 4]: byte (g, m, i) belongs to features
    ``128 g + 32 i`` .. ``+ 31`` of row m.  ``shape`` is x's; its leading
    dimensions make up the M rows."""
    codes: torch.Tensor
    scales: torch.Tensor
    shape: tuple[int, ...]
    dtype: torch.dtype

    @property
    def device(self):
        return self.codes.device

    @property
    def rows(self) -> int:
        n = 1
        for d in self.shape[:-1]:
            n *= d
        return n

    def nbytes(self) -> int:
        return self.codes.numel() + self.scales.numel()

    def check(self) -> None:
        """Raises unless the tensors have the layout the kernels read."""
        codes, scales = self.codes, self.scales
        M, K = self.rows, self.shape[-1]
        if codes.dtype != torch.int8 or codes.shape != (M, K):
            raise ShapeError(f"checkpoint codes must be int8 {(M, K)}, got "
                             f"{tuple(codes.shape)} {codes.dtype}")
        want = (-(-K // 128), -(-M // 4) * 4, 4)
        if scales.dtype != torch.uint8 or scales.shape != want or not scales.is_contiguous():
            raise ShapeError(f"checkpoint scales must be contiguous uint8 {want}, got "
                             f"{tuple(scales.shape)} {scales.dtype}")
        ld, one = codes.stride()
        if M and (one != 1 or ld < K or ld % 16):
            raise ShapeError("checkpoint code rows must be contiguous and a multiple of 16 bytes "
                             f"apart, got strides {(ld, one)}")
        if scales.device != codes.device:
            raise DeviceError("checkpoint codes and scales are on different devices")

    def dequantize(self, dtype: torch.dtype | None = None) -> torch.Tensor:
        """The values, shaped as x, in ``dtype`` (default: x's; exact in bf16)."""
        self.check()
        _need_cuda(self.codes)
        _need_current(self.codes)
        out = self.codes.new_empty(self.shape, dtype=dtype or self.dtype)
        if out.numel():
            st = _lib.load().mlora_act_restore(_ptr(self.codes), self.codes.stride(0),
                                               _ptr(self.scales), self.rows, self.shape[-1],
                                               _ptr(out), _dtype_code(out), _stream())
            _lib.check(st, "mlora_act_restore")
        return out


def empty_checkpoint(like: torch.Tensor) -> ActivationCheckpoint:
    """An uninitialised checkpoint of activations like these: the buffers a
    forward fills (``kernels.lora_linear_fwd(..., ckpt_out=)``)."""
    shape = tuple(like.shape)
    if not shape or shape[-1] == 0:
        raise ShapeError("a checkpoint is of activations with at least one feature")
    K, M = shape[-1], 1
    for d in shape[:-1]:
        M *= d
    ld = -(-K // 16) * 16
    codes = like.new_empty((M, ld), dtype=torch.int8)
    scales = like.new_empty((-(-K // 128), -(-M // 4) * 4, 4), dtype=torch.uint8)
    return ActivationCheckpoint(codes if ld == K else codes[:, :K], scales, shape, like.dtype)


def checkpoint_activation(x: torch.Tensor) -> ActivationCheckpoint:
    """Quantises activations [..., K] (bf16/fp16/fp32) to MXINT8.  Layers that
    share an input can share one checkpoint: ``c = checkpoint_activation(x)``,
    then ``q_proj(x, checkpoint=c)``, ``k_proj(x, checkpoint=c)``, ..."""
    _need_cuda(x)
    _need_current(x)
    code = _dtype_code(x)
    c = empty_checkpoint(x)
    M, K = c.codes.shape
    if M:
        if not x.is_contiguous():
            x = x.detach().contiguous()
        st = _lib.load().mlora_act_checkpoint(x.data_ptr(), code, M, K, c.codes.data_ptr(),
                                              c.codes.stride(0), c.scales.data_ptr(), _stream())
        _lib.check(st, "mlora_act_checkpoint")
    return c


# ------------------------------------------------------------ pack format --
# The reference has no on-disk form for a quantised base.  This one keeps the
# kernels' layout unchanged: one safetensors file holding, per weight,
# ``{name}.codes`` (uint8), ``{name}.scales`` (fp32 absmax for NF4, fp16 for
# INT4/INT8, uint8 for MXFP4) and, for INT4/INT8, ``{name}.zeros`` (fp16); the safetensors
# header metadata carries ``format`` = PACK_FORMAT and ``weights`` = a JSON map
# name -> {scheme, group, out_features, in_features}.  Files written here load
# without any conversion and are validated shape by shape on load.

PACK_FORMAT = "metallora-qbase-1"


def _expected_shapes(scheme: str, N: int, K: int, group: int):
    per_byte = 1 if scheme == "int8" else 2
    groups = -(-K // group)
    codes = (N, -(-K // per_byte))
    return codes, (N, groups), _SCALE_DTYPE[scheme]


def pack_quantized(weights: dict[str, QuantizedWeight]) -> tuple[dict, dict]:
    """(tensors, metadata) of the pack format for ``{name: QuantizedWeight}``;
    tensors are copied to host memory."""
    tensors: dict[str, torch.Tensor] = {}
    meta = {}
    for name, qw in weights.items():
        tensors[f"{name}.codes"] = qw.codes.detach().contiguous().cpu()
        tensors[f"{name}.scales"] = qw.scales.detach().contiguous().cpu()
        if qw.zeros is not None:
            tensors[f"{name}.zeros"] = qw.zeros.detach().contiguous().cpu()
        meta[name] = {"scheme": qw.scheme, "group": int(qw.group),
                      "out_features": int(qw.shape[0]), "in_features": int(qw.shape[1])}
    import json
    return tensors, {"format": PACK_FORMAT, "weights": json.dumps(meta, sort_keys=True)}


def unpack_quantized(tensors: dict, metadata: dict, device=None,
                     lean: bool = False) -> dict[str, QuantizedWeight]:
    """Inverse of ``pack_quantized``; every tensor is checked against the
    shape and dtype its scheme, group and weight shape imply."""
    import json
    if (metadata or {}).get("format") != PACK_FORMAT:
        raise QuantizationError(f"not a {PACK_FORMAT} pack (metadata {metadata!r})")
    out = {}
    for name, m in json.loads(metadata["weights"]).items():
        scheme, group = m["scheme"], int(m["group"])
        N, K = int(m["out_features"]), int(m["in_features"])
        if scheme not in SCHEMES:
            raise QuantizationError(f"{name}: unknown scheme {scheme!r}")
        codes_shape, scales_shape, scale_dt = _expected_shapes(scheme, N, K, group)
        want = {"codes": (codes_shape, torch.uint8), "scales": (scales_shape, scale_dt)}
        if scheme in _WITH_ZEROS:
            want["zeros"] = (scales_shape, torch.float16)
        got = {}
        for part, (shape, dt) in want.items():
            t = tensors.get(f"{name}.{part}")
            if t is None:
                raise QuantizationError(f"{name}: missing {part}")
            if tuple(t.shape) != shape or t.dtype != dt:
                raise QuantizationError(f"{name}.{part}: expected {shape} {dt}, got "
                                        f"{tuple(t.shape)} {t.dtype}")
            got[part] = t.to(device) if device is not None else t
        out[name] = from_reference_layout(scheme, got["codes"], got["scales"], got.get("zeros"),
                                          (N, K), group, lean=lean)
    return out


def save_quantized(weights: dict[str, QuantizedWeight], path) -> None:
    """Writes ``{name: QuantizedWeight}`` to one safetensors file in the pack format."""
    from safetensors.torch import save_file
    tensors, meta = pack_quantized(weights)
    save_file(tensors, str(path), metadata=meta)


def load_quantized(path, device=None, lean: bool = False) -> dict[str, QuantizedWeight]:
    """Reads a pack written by ``save_quantized`` (onto ``device`` if given)."""
    from safetensors import safe_open
    tensors = {}
    with safe_open(str(path), framework="pt") as f:
        meta = f.metadata()
        for k in f.keys():
            tensors[k] = f.get_tensor(k)
    return unpack_quantized(tensors, meta, device=device, lean=lean)
