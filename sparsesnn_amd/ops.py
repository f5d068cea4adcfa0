"""Torch-facing wrappers over the C ABI of libsengine_amd.so.

PyTorch is used for device memory and the current stream only; every op launches a
hand-written gfx950 HIP kernel and there is no fallback path.  Each wrapper checks the
tensors against the descriptor on the host before launching (the C ABI takes raw
pointers and cannot check buffer sizes itself).
"""
from __future__ import annotations

import ctypes
import math
import os
from dataclasses import dataclass, replace
from typing import Optional

import torch
from torch.autograd import forward_ad

from . import _lib
from ._lib import (ACTIVATIONS, ENC_BF16, ENC_BITS, ENC_E4M3, ENC_F16, ENC_F32, NEURON_IF, NEURON_LIF, NEURON_MS,
                   WLAYOUT_HWIO, WLAYOUT_OIHW, ConvLifDesc, CrossDesc, DecayDesc, LinearDesc, LinearE2m1Desc, RmsNormDesc,
                   RotaryDesc, SEngineError, check)

__all__ = [
    "ConvSpec", "make_desc", "geometry", "set_fused_kernel", "compress_2_4", "pack_dense_weights", "pack_spikes",
    "unpack_spikes", "fused_sparse_conv_bn_lif", "fused_sparse_conv_bn_lif_add", "stem_conv_bn",
    "multistep_neuron_repeat", "maxpool_spikes", "sew_head", "dense_conv_bn", "multistep_neuron", "SEngineError",
    "ENC_BITS", "ENC_F16", "ENC_F32", "NEURON_LIF", "NEURON_IF", "NEURON_MS", "WLAYOUT_OIHW", "WLAYOUT_HWIO",
    "neuron_code", "fused_sparse_conv_bn_add_neuron", "spiking_self_attention", "stem_conv_bn_neuron",
    "fused_sparse_conv_bn_lif_pair", "fused_sparse_conv_bn_lif_split", "fused_sparse_conv_bn_lif_tail", "tail_eligible",
    "fused_plan", "rms_norm", "linear", "cross_attention", "rotary", "linear_e2m1", "decay_attention",
    "ENC_BF16", "ENC_E4M3",
]


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)  # absent in CPU-only builds


def _stream(device: torch.device):
    """The device's current stream as an integer handle (no torch Stream object is made)."""
    if _raw_stream is not None and device.index is not None:
        return _raw_stream(device.index)
    return torch.cuda.current_stream(device).cuda_stream


def _fits(t, dtype: torch.dtype, numel: int) -> bool:
    """Whether _require_cuda and _require_numel both accept t."""
    return isinstance(t, torch.Tensor) and t.is_cuda and t.dtype is dtype and t.numel() == numel and t.is_contiguous()


def _require_cuda(t: torch.Tensor, name: str):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if t.device.type != "cuda":
        raise SEngineError(f"{name} must be on a HIP device (got {t.device})")
    if not t.is_contiguous():
        raise SEngineError(f"{name} must be contiguous")


def _require_numel(t: torch.Tensor, n: int, dtype, name: str):
    if t.dtype != dtype:
        raise SEngineError(f"{name}: expected dtype {dtype}, got {t.dtype}")
    if t.numel() != n:
        raise SEngineError(f"{name}: expected {n} elements, got {t.numel()}")


@dataclass(frozen=True)
class ConvSpec:
    """Shape + neuron parameters of one Conv+BN+neuron node (ConvParams + NeuronParams,
    sengine/ir.py:179-201, plus the T/B extents the reference bakes into each kernel)."""

    T: int
    B: int
    C_in: int
    H: int
    W: int
    C_out: int
    KH: int = 3
    KW: int = 3
    stride: int = 1
    padding: int = 1
    dilation: int = 1
    neuron: str = "lif"          # "lif" | "if" | "ms" (MS-ResNet neuron: `tau` holds its decay)
    hard_reset: bool = True
    tau: float = 2.0
    v_threshold: float = 1.0
    v_reset: float = 0.0
    in_enc: int = ENC_BITS
    out_enc: int = ENC_BITS
    weight_planes: int = 1

    def desc(self) -> ConvLifDesc:
        return make_desc(self)

    def __getstate__(self):
        """The fields alone: what is derived from them (ctypes objects) is rebuilt where it is needed."""
        return {k: v for k, v in self.__dict__.items() if not k.startswith("_")}

    def with_enc(self, in_enc: int, out_enc: int) -> "ConvSpec":
        """This spec with other encodings; made once per pair and kept, with its own plan."""
        made = self.__dict__.get("_variants")
        if made is None:
            made = {}
            object.__setattr__(self, "_variants", made)
        v = made.get((in_enc, out_enc))
        if v is None:
            v = made[(in_enc, out_enc)] = replace(self, in_enc=in_enc, out_enc=out_enc)
        return v


def _ref(s: ConvSpec):
    """The spec's C descriptor by reference (which keeps it alive), made once per spec."""
    r = s.__dict__.get("_desc_ref")
    if r is None:
        r = ctypes.byref(make_desc(s))
        object.__setattr__(s, "_desc_ref", r)
    return r


class _Plan:
    """What every call derives from a ConvSpec alone: its C descriptor, geometry, blob sizes and
    activation layouts.  A spec is immutable, so they are worked out once and kept on it (a call
    spent more host time on them than on its launch)."""

    __slots__ = ("ref", "OH", "OW", "M", "_blob", "_dense", "_in", "_out")

    def __init__(self, s: "ConvSpec"):
        lib = _lib.load()
        self.ref = _ref(s)
        oh, ow = ctypes.c_int32(), ctypes.c_int32()
        m, k = ctypes.c_int64(), ctypes.c_int64()
        check(lib.sengine_amd_conv_geometry(self.ref, ctypes.byref(oh), ctypes.byref(ow), ctypes.byref(m),
                                            ctypes.byref(k)), "conv_geometry")
        self.OH, self.OW, self.M = oh.value, ow.value, m.value
        self._blob = self._dense = self._in = self._out = None

    def blob(self):
        """(value bytes, metadata bytes) of the sparse weight blob."""
        if self._blob is None:
            vb, mb = ctypes.c_size_t(), ctypes.c_size_t()
            check(_lib.load().sengine_amd_sparse_blob_bytes(self.ref, ctypes.byref(vb), ctypes.byref(mb)),
                  "sparse_blob_bytes")
            self._blob = (vb.value, mb.value)
        return self._blob

    def dense_blob(self) -> int:
        if self._dense is None:
            vb = ctypes.c_size_t()
            check(_lib.load().sengine_amd_dense_blob_bytes(self.ref, ctypes.byref(vb)), "dense_blob_bytes")
            self._dense = vb.value
        return self._dense

    def data(self, s: "ConvSpec"):
        """(dtype, numel) of the input."""
        if self._in is None:
            self._in = _enc_numel(s.in_enc, s.T * s.B * s.H * s.W * s.C_in)
        return self._in

    def spikes(self, s: "ConvSpec"):
        """(dtype, numel, shape) of the output spikes."""
        if self._out is None:
            dt, n = _enc_numel(s.out_enc, s.T * self.M * s.C_out)
            last = s.C_out // 32 if s.out_enc == ENC_BITS else s.C_out
            self._out = (dt, n, (s.T * s.B, self.OH, self.OW, last))
        return self._out


def _plan(s: ConvSpec) -> _Plan:
    p = s.__dict__.get("_plan")
    if p is None:
        p = _Plan(s)
        object.__setattr__(s, "_plan", p)
    return p


def _check_fused(who: str, s: ConvSpec, p: _Plan, data, values, meta, bn_scale, bn_bias, extra=()):
    """The checks shared by the fused calls: the input and the weight blob against the descriptor,
    the BN vectors, and `extra` tensors that only have to be contiguous on the device."""
    vb, mb = p.blob()
    dt, n_in = p.data(s) if isinstance(data, torch.Tensor) and data.is_cuda else (None, 0)
    if _fits(data, dt, n_in) and _fits(bn_scale, torch.float32, s.C_out) and _fits(bn_bias, torch.float32, s.C_out) \
            and isinstance(values, torch.Tensor) and values.is_cuda and values.is_contiguous() and values.nbytes == vb \
            and isinstance(meta, torch.Tensor) and meta.is_cuda and meta.is_contiguous() and meta.nbytes == mb \
            and all(isinstance(t, torch.Tensor) and t.is_cuda and t.is_contiguous() for t, _ in extra):
        return
    for t, n in ((data, "data"), (values, "values"), (meta, "meta"), (bn_scale, "bn_scale"), (bn_bias, "bn_bias"),
                 *extra):
        _require_cuda(t, n)
    dt, n_in = p.data(s)
    _require_numel(data, n_in, dt, "data")
    if values.numel() * values.element_size() != vb or meta.numel() * meta.element_size() != mb:
        raise SEngineError(f"{who}: weight blob does not match the descriptor")
    _require_numel(bn_scale, s.C_out, torch.float32, "bn_scale")
    _require_numel(bn_bias, s.C_out, torch.float32, "bn_bias")


def _check_req(t, numel: int, dtype: torch.dtype, name: str):
    if not _fits(t, dtype, numel):
        _require_cuda(t, name)
        _require_numel(t, numel, dtype, name)


def _check_opt(t, numel: int, dtype: torch.dtype, name: str):
    """An optional buffer of a call (None passes)."""
    if t is not None:
        _check_req(t, numel, dtype, name)


_NEURON_CODES = {"lif": NEURON_LIF, "if": NEURON_IF, "ms": NEURON_MS}


def neuron_code(name: str) -> int:
    """C-ABI neuron kind for 'lif' | 'if' | 'ms'."""
    if name not in _NEURON_CODES:
        raise ValueError(f"neuron must be 'lif', 'if' or 'ms', got {name!r}")
    return _NEURON_CODES[name]


def make_desc(s: ConvSpec) -> ConvLifDesc:
    return ConvLifDesc(
        T=s.T, B=s.B, C_in=s.C_in, H=s.H, W=s.W, C_out=s.C_out, KH=s.KH, KW=s.KW,
        stride_h=s.stride, stride_w=s.stride, pad_h=s.padding, pad_w=s.padding,
        dil_h=s.dilation, dil_w=s.dilation,
        neuron=neuron_code(s.neuron), hard_reset=int(bool(s.hard_reset)),
        tau=float(s.tau), v_threshold=float(s.v_threshold), v_reset=float(s.v_reset),
        in_enc=s.in_enc, out_enc=s.out_enc, weight_planes=s.weight_planes)


def set_fused_kernel(choice: str) -> None:
    """Kernel for spike-bit inputs: 'auto' (split-K small-M kernel for small outputs, else the
    halo-tiled kernel where eligible, else the LDS-staged kernel), 'direct' (direct-gather
    kernel), 'lds' (LDS-staged kernel) or 'tile' (halo-tiled kernel where eligible)."""
    lib = _lib.load()
    check(lib.sengine_amd_set_fused_kernel({"auto": 0, "direct": 1, "lds": 2, "tile": 3}[choice]),
          "set_fused_kernel")


PLAN_TRACES, PLAN_STATE, PLAN_SEW_ADD, PLAN_SHORTCUT, PLAN_TAIL = 1, 2, 4, 8, 16


def fused_plan(s: ConvSpec, traces: bool = False, state: bool = False, sew_add: bool = False,
               shortcut: bool = False, tail: bool = False) -> str:
    """Name of the kernel instance a fused call with these optional buffers would launch
    (route and compile-time specialisation); tail: the paired-tail call
    (fused_sparse_conv_bn_lif_tail).  Host-only, launches nothing."""
    lib = _lib.load()
    d = make_desc(s)
    flags = ((PLAN_TRACES if traces else 0) | (PLAN_STATE if state else 0) | (PLAN_SEW_ADD if sew_add else 0)
             | (PLAN_SHORTCUT if shortcut else 0) | (PLAN_TAIL if tail else 0))
    buf = ctypes.create_string_buffer(256)
    check(lib.sengine_amd_fused_plan(ctypes.byref(d), flags, buf, len(buf)), "fused_plan")
    return buf.value.decode()


def geometry(s: ConvSpec):
    """(OH, OW, M_per_t, K_red) of a node."""
    lib = _lib.load()
    d = make_desc(s)
    oh, ow = ctypes.c_int32(), ctypes.c_int32()
    m, k = ctypes.c_int64(), ctypes.c_int64()
    check(lib.sengine_amd_conv_geometry(ctypes.byref(d), ctypes.byref(oh), ctypes.byref(ow),
                                        ctypes.byref(m), ctypes.byref(k)), "conv_geometry")
    return oh.value, ow.value, m.value, k.value


def _enc_numel(enc: int, n_values: int) -> tuple:
    """(dtype, numel) of a tensor holding n_values activations in encoding enc."""
    if enc == ENC_BITS:
        if n_values % 32:
            raise SEngineError("bit-encoded tensors need a multiple of 32 values")
        return torch.int32, n_values // 32
    if enc == ENC_F16:
        return torch.float16, n_values
    if enc == ENC_F32:
        return torch.float32, n_values
    raise SEngineError(f"unknown encoding {enc}")


def _weight_enc(w: torch.Tensor) -> int:
    if w.dtype == torch.float32:
        return ENC_F32
    if w.dtype == torch.float16:
        return ENC_F16
    raise SEngineError(f"weights must be fp32 or fp16, got {w.dtype}")


def _check_weight(s: ConvSpec, w: torch.Tensor, layout: int):
    _require_cuda(w, "weight")
    shape = (s.C_out, s.C_in, s.KH, s.KW) if layout == WLAYOUT_OIHW else (s.KH, s.KW, s.C_in, s.C_out)
    if tuple(w.shape) != shape:
        raise SEngineError(f"weight: expected shape {shape}, got {tuple(w.shape)}")


def _blob_bytes(lib, d, tail: bool):
    vb, mb = ctypes.c_size_t(), ctypes.c_size_t()
    if tail:
        check(lib.sengine_amd_tail_blob_bytes(ctypes.byref(d), ctypes.byref(vb), ctypes.byref(mb)), "tail_blob_bytes")
    else:
        check(lib.sengine_amd_sparse_blob_bytes(ctypes.byref(d), ctypes.byref(vb), ctypes.byref(mb)),
              "sparse_blob_bytes")
    return vb, mb


def compress_2_4(s: ConvSpec, weight: torch.Tensor, layout: int = WLAYOUT_OIHW, check_pattern: bool = True,
                 tail: bool = False):
    """2:4-compress a conv weight on the GPU -> (values int16 tensor, meta int32 tensor, violations).

    Raises if check_pattern and any 4-group along C_in holds more than two entries with
    |w| >= 1e-10 (such weights belong on the dense fallback, sengine/optimizer.py:845-853).
    tail: the blob of the paired-tail call (fused_sparse_conv_bn_lif_tail), for a 3x3 conv
    whose last 32 input channels are zero padding; a nonzero weight there is a violation."""
    lib = _lib.load()
    _check_weight(s, weight, layout)
    d = make_desc(s)
    vb, mb = _blob_bytes(lib, d, tail)
    dev = weight.device
    values = torch.empty(vb.value // 2, dtype=torch.int16, device=dev)
    meta = torch.empty(mb.value // 4, dtype=torch.int32, device=dev)
    n_groups = lib.sengine_amd_num_groups(ctypes.byref(d))
    # zeroed: in the flat (small-output) layout taps that never touch the image are not visited
    viol = torch.zeros(n_groups, dtype=torch.int32, device=dev)
    fn = lib.sengine_amd_compress_2_4_tail if tail else lib.sengine_amd_compress_2_4
    check(fn(ctypes.byref(d), _ptr(weight), _weight_enc(weight), layout, _ptr(values), _ptr(meta), _ptr(viol),
             _stream(dev)), "compress_2_4")
    if check_pattern:
        n_bad = int(viol.sum().item())
        if n_bad:
            raise SEngineError(f"compress_2_4: {n_bad} 4-groups have more than two non-zero weights"
                               + (" or a nonzero weight in the last 32 (padding) input channels" if tail else ""))
    return values, meta, viol


def pack_dense_weights(s: ConvSpec, weight: torch.Tensor, layout: int = WLAYOUT_OIHW) -> torch.Tensor:
    lib = _lib.load()
    _check_weight(s, weight, layout)
    d = make_desc(s)
    vb = ctypes.c_size_t()
    check(lib.sengine_amd_dense_blob_bytes(ctypes.byref(d), ctypes.byref(vb)), "dense_blob_bytes")
    values = torch.empty(vb.value // 2, dtype=torch.int16, device=weight.device)
    check(lib.sengine_amd_pack_dense_weights(ctypes.byref(d), _ptr(weight), _weight_enc(weight), layout,
                                             _ptr(values), _stream(weight.device)), "pack_dense_weights")
    return values


def pack_spikes(x: torch.Tensor, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Dense (..., C) fp16/fp32 -> spike bits int32 (..., C/32) (value != 0 -> 1)."""
    lib = _lib.load()
    _require_cuda(x, "x")
    C = x.shape[-1]
    if C % 32:
        raise SEngineError("pack_spikes: last dim must be a multiple of 32")
    enc = ENC_F16 if x.dtype == torch.float16 else ENC_F32 if x.dtype == torch.float32 else None
    if enc is None:
        raise SEngineError("pack_spikes: x must be fp16 or fp32")
    n_pos = x.numel() // C
    if out is None:
        out = torch.empty(*x.shape[:-1], C // 32, dtype=torch.int32, device=x.device)
    else:
        _require_cuda(out, "out")
        _require_numel(out, n_pos * (C // 32), torch.int32, "out")
    check(lib.sengine_amd_pack_spikes(_ptr(x), enc, n_pos, C, _ptr(out), _stream(x.device)), "pack_spikes")
    return out


def unpack_spikes(bits: torch.Tensor, C: int, dtype=torch.float16, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    lib = _lib.load()
    _require_cuda(bits, "bits")
    if C % 32 or bits.shape[-1] != C // 32 or bits.dtype != torch.int32:
        raise SEngineError("unpack_spikes: bits must be int32 (..., C/32)")
    enc = ENC_F16 if dtype == torch.float16 else ENC_F32 if dtype == torch.float32 else None
    if enc is None:
        raise SEngineError("unpack_spikes: dtype must be fp16 or fp32")
    n_pos = bits.numel() // (C // 32)
    if out is None:
        out = torch.empty(*bits.shape[:-1], C, dtype=dtype, device=bits.device)
    else:
        _require_cuda(out, "out")
        _require_numel(out, n_pos * C, dtype, "out")
    check(lib.sengine_amd_unpack_spikes(_ptr(bits), n_pos, C, _ptr(out), enc, _stream(bits.device)), "unpack_spikes")
    return out


def fused_sparse_conv_bn_lif(s: ConvSpec, data: torch.Tensor, values: torch.Tensor, meta: torch.Tensor,
                             bn_scale: torch.Tensor, bn_bias: torch.Tensor, state: Optional[torch.Tensor] = None,
                             out: Optional[torch.Tensor] = None, h_trace: Optional[torch.Tensor] = None,
                             x_trace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Fused 2:4 Conv + BN + multi-step neuron (one launch).  Returns the spike tensor:
    bits int32 (T*B, OH, OW, C_out/32) or fp16 (T*B, OH, OW, C_out) per s.out_enc."""
    lib = _lib.load()
    p = _plan(s)
    _check_fused("fused_sparse_conv_bn_lif", s, p, data, values, meta, bn_scale, bn_bias)
    dev = data.device
    _check_opt(state, p.M * s.C_out, torch.float32, "state")
    _check_opt(h_trace, s.T * p.M * s.C_out, torch.float32, "h_trace")
    _check_opt(x_trace, s.T * p.M * s.C_out, torch.float32, "x_trace")
    odt, n_out, shape = p.spikes(s)
    if out is None:
        out = torch.empty(shape, dtype=odt, device=dev)
    else:
        _check_opt(out, n_out, odt, "out")
    check(lib.sengine_amd_fused_sparse_conv_bn_lif(
        p.ref, data.data_ptr(), values.data_ptr(), meta.data_ptr(), _ptr(state), bn_scale.data_ptr(),
        bn_bias.data_ptr(), out.data_ptr(), _ptr(h_trace), _ptr(x_trace), _stream(dev)), "fused_sparse_conv_bn_lif")
    return out


def tail_eligible(spec: ConvSpec, in_channels_real) -> bool:
    """Whether a fused 3x3 node whose last 32 input channels are zero padding runs the paired-tail
    call (fused_sparse_conv_bn_lif_tail: the last chunk's 32 real channels of two taps per
    reduction step) -- opt-in, SENGINE_AMD_TAIL=1 (read when an engine is built), where the
    shape and neuron allow it: it does 22 % fewer SMFMACs but runs on the persistent 3x3 kernel,
    which measured slower on such multi-chunk layers than the ordinary call over the padded
    blob (Spikformer's proj_conv2: 1,234-1,248 us against 1,192)."""
    return (os.environ.get("SENGINE_AMD_TAIL", "0") == "1" and in_channels_real is not None and int(in_channels_real) == spec.C_in - 32 and spec.KH == 3
            and spec.KW == 3 and spec.stride == 1 and spec.padding == 1 and spec.dilation == 1 and spec.T == 4
            and spec.weight_planes == 1 and spec.hard_reset and spec.v_reset == 0.0
            and (spec.neuron == "if" or (spec.neuron == "lif" and math.log2(spec.tau).is_integer())))


def fused_sparse_conv_bn_lif_tail(s: ConvSpec, data: torch.Tensor, values: torch.Tensor, meta: torch.Tensor,
                                  bn_scale: torch.Tensor, bn_bias: torch.Tensor, state: Optional[torch.Tensor] = None,
                                  out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The paired-tail fused call: a 3x3 conv whose last 32 input channels are zero padding, with
    the blob of compress_2_4(..., tail=True); spike bits in and out, T = 4, no traces.  Returns
    the spike bits int32 (T*B, OH, OW, C_out/32)."""
    lib = _lib.load()
    OH, OW, M, _ = geometry(s)
    d = make_desc(s)
    vb, mb = _blob_bytes(lib, d, True)
    for t, n in ((data, "data"), (values, "values"), (meta, "meta"), (bn_scale, "bn_scale"), (bn_bias, "bn_bias")):
        _require_cuda(t, n)
    dt, n_in = _enc_numel(s.in_enc, s.T * s.B * s.H * s.W * s.C_in)
    _require_numel(data, n_in, dt, "data")
    if values.numel() * values.element_size() != vb.value or meta.numel() * meta.element_size() != mb.value:
        raise SEngineError("fused_sparse_conv_bn_lif_tail: weight blob does not match the descriptor")
    _require_numel(bn_scale, s.C_out, torch.float32, "bn_scale")
    _require_numel(bn_bias, s.C_out, torch.float32, "bn_bias")
    if state is not None:
        _require_cuda(state, "state")
        _require_numel(state, M * s.C_out, torch.float32, "state")
    odt, n_out = _enc_numel(s.out_enc, s.T * M * s.C_out)
    if out is None:
        out = torch.empty(s.T * s.B, OH, OW, s.C_out // 32, dtype=odt, device=data.device)
    else:
        _require_cuda(out, "out")
        _require_numel(out, n_out, odt, "out")
    check(lib.sengine_amd_fused_sparse_conv_bn_lif_tail(ctypes.byref(d), _ptr(data), _ptr(values), _ptr(meta),
                                                        _ptr(state), _ptr(bn_scale), _ptr(bn_bias), _ptr(out),
                                                        _stream(data.device)), "fused_sparse_conv_bn_lif_tail")
    return out


def fused_sparse_conv_bn_lif_split(s: ConvSpec, data: torch.Tensor, values: torch.Tensor, meta: torch.Tensor,
                                   bn_scale: torch.Tensor, bn_bias: torch.Tensor, split: int,
                                   out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """fused_sparse_conv_bn_lif with the spike bits split by channel into planes of `split`
    channels (layers concatenated along C_out that read the same input): returns int32
    (ceil(C_out / split), T*B, OH, OW, split/32); plane k holds channels [k*split, (k+1)*split)."""
    lib = _lib.load()
    if s.out_enc != ENC_BITS:
        raise SEngineError("fused_sparse_conv_bn_lif_split: spike-bit output only")
    p = _plan(s)
    _check_fused("fused_sparse_conv_bn_lif_split", s, p, data, values, meta, bn_scale, bn_bias)
    nplanes = -(-s.C_out // split)
    if out is None:
        out = torch.empty(nplanes, s.T * s.B, p.OH, p.OW, split // 32, dtype=torch.int32, device=data.device)
    else:
        _check_opt(out, nplanes * s.T * p.M * split // 32, torch.int32, "out")
    check(lib.sengine_amd_fused_sparse_conv_bn_lif_split(
        p.ref, _ptr(data), _ptr(values), _ptr(meta), None, _ptr(bn_scale), _ptr(bn_bias), _ptr(out), split,
        _stream(data.device)), "fused_sparse_conv_bn_lif_split")
    return out


def fused_sparse_conv_bn_lif_pair(s0: ConvSpec, s1: ConvSpec, data: torch.Tensor, values0: torch.Tensor,
                                  meta0: torch.Tensor, bn_scale0: torch.Tensor, bn_bias0: torch.Tensor,
                                  values1: torch.Tensor, meta1: torch.Tensor, bn_scale1: torch.Tensor,
                                  bn_bias1: torch.Tensor, out0: Optional[torch.Tensor] = None,
                                  out1: Optional[torch.Tensor] = None):
    """Two fused 2:4 Conv + BN + neuron nodes on the same input (a block's conv1 and its
    downsample), one launch where both run on the small-output kernel.  Returns (out0, out1),
    each as fused_sparse_conv_bn_lif would."""
    lib = _lib.load()
    for s in (s0, s1):
        if (s.T, s.B, s.C_in, s.H, s.W, s.in_enc) != (s0.T, s0.B, s0.C_in, s0.H, s0.W, s0.in_enc):
            raise SEngineError("fused_sparse_conv_bn_lif_pair: the two convs must read the same input")
    dev = data.device
    dt, n_in = _enc_numel(s0.in_enc, s0.T * s0.B * s0.H * s0.W * s0.C_in)
    _require_cuda(data, "data")
    _require_numel(data, n_in, dt, "data")
    outs = []
    for s, values, meta, sc, bi, out, tag in ((s0, values0, meta0, bn_scale0, bn_bias0, out0, "0"),
                                               (s1, values1, meta1, bn_scale1, bn_bias1, out1, "1")):
        OH, OW, M, _ = geometry(s)
        d = make_desc(s)
        vb, mb = ctypes.c_size_t(), ctypes.c_size_t()
        check(lib.sengine_amd_sparse_blob_bytes(ctypes.byref(d), ctypes.byref(vb), ctypes.byref(mb)),
              "sparse_blob_bytes")
        for t, n in ((values, "values"), (meta, "meta"), (sc, "bn_scale"), (bi, "bn_bias")):
            _require_cuda(t, n + tag)
        if values.numel() * values.element_size() != vb.value or meta.numel() * meta.element_size() != mb.value:
            raise SEngineError(f"fused_sparse_conv_bn_lif_pair: weight blob {tag} does not match its descriptor")
        _require_numel(sc, s.C_out, torch.float32, "bn_scale" + tag)
        _require_numel(bi, s.C_out, torch.float32, "bn_bias" + tag)
        odt, n_out = _enc_numel(s.out_enc, s.T * M * s.C_out)
        if out is None:
            last = s.C_out // 32 if s.out_enc == ENC_BITS else s.C_out
            out = torch.empty(s.T * s.B, OH, OW, last, dtype=odt, device=dev)
        else:
            _require_cuda(out, "out" + tag)
            _require_numel(out, n_out, odt, "out" + tag)
        outs.append(out)
    d0, d1 = make_desc(s0), make_desc(s1)
    check(lib.sengine_amd_fused_sparse_conv_bn_lif_pair(
        ctypes.byref(d0), ctypes.byref(d1), _ptr(data), _ptr(values0), _ptr(meta0), _ptr(bn_scale0), _ptr(bn_bias0),
        _ptr(outs[0]), _ptr(values1), _ptr(meta1), _ptr(bn_scale1), _ptr(bn_bias1), _ptr(outs[1]), _stream(dev)),
        "fused_sparse_conv_bn_lif_pair")
    return outs[0], outs[1]


def fused_sparse_conv_bn_lif_add(s: ConvSpec, data: torch.Tensor, values: torch.Tensor, meta: torch.Tensor,
                                 bn_scale: torch.Tensor, bn_bias: torch.Tensor, residual: torch.Tensor,
                                 residual_planes: int, out_planes: int, state: Optional[torch.Tensor] = None,
                                 out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Fused 2:4 Conv + BN + neuron + SEW 'ADD' residual: out = spike + residual as
    `out_planes` bit planes, int32 (T*B, OH, OW, out_planes*C_out/32).  With s.out_enc ==
    ENC_F16, out is fp16 (T*B, OH, OW, C_out) and the residual fp16 of that shape
    (residual_planes == 0) or `residual_planes` bit planes; out_planes is unused."""
    lib = _lib.load()
    f16 = s.out_enc == ENC_F16
    if s.out_enc != ENC_BITS and not f16:
        raise SEngineError("fused_sparse_conv_bn_lif_add: out_enc must be ENC_BITS or ENC_F16")
    p = _plan(s)
    _check_fused("fused_sparse_conv_bn_lif_add", s, p, data, values, meta, bn_scale, bn_bias,
                 extra=((residual, "residual"),))
    M, dev = p.M, data.device
    if f16 and residual_planes == 0:
        out_planes = 0
        _require_numel(residual, s.T * M * s.C_out, torch.float16, "residual")
    else:
        _require_numel(residual, s.T * M * residual_planes * s.C_out // 32, torch.int32, "residual")
    _check_opt(state, M * s.C_out, torch.float32, "state")
    if out is None:
        out = (torch.empty((s.T * s.B, p.OH, p.OW, s.C_out), dtype=torch.float16, device=dev) if f16 else
               torch.empty((s.T * s.B, p.OH, p.OW, out_planes * s.C_out // 32), dtype=torch.int32, device=dev))
    elif f16:
        _check_opt(out, s.T * M * s.C_out, torch.float16, "out")
    else:
        _check_opt(out, s.T * M * out_planes * s.C_out // 32, torch.int32, "out")
    check(lib.sengine_amd_fused_sparse_conv_bn_lif_add(
        p.ref, _ptr(data), _ptr(values), _ptr(meta), _ptr(state), _ptr(bn_scale), _ptr(bn_bias), _ptr(residual),
        int(residual_planes), _ptr(out), int(out_planes), _stream(dev)), "fused_sparse_conv_bn_lif_add")
    return out


def fused_sparse_conv_bn_add_neuron(s: ConvSpec, data: torch.Tensor, values: torch.Tensor, meta: torch.Tensor,
                                    bn_scale: torch.Tensor, bn_bias: torch.Tensor,
                                    residual: Optional[torch.Tensor] = None, state: Optional[torch.Tensor] = None,
                                    real_out: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None):
    """Membrane-shortcut form (MS-ResNet): y = BN(conv(data)) + residual (fp32 NHWC
    (T*B, OH, OW, C_out), or none) and the neuron of `s` run over y.  Returns (y, spikes)."""
    lib = _lib.load()
    p = _plan(s)
    _check_fused("fused_sparse_conv_bn_add_neuron", s, p, data, values, meta, bn_scale, bn_bias)
    dev = data.device
    n_real = s.T * p.M * s.C_out
    _check_opt(residual, n_real, torch.float32, "residual")
    _check_opt(state, p.M * s.C_out, torch.float32, "state")
    if real_out is None:
        real_out = torch.empty((s.T * s.B, p.OH, p.OW, s.C_out), dtype=torch.float32, device=dev)
    else:
        _check_opt(real_out, n_real, torch.float32, "real_out")
    odt, n_out, shape = p.spikes(s)
    if out is None:
        out = torch.empty(shape, dtype=odt, device=dev)
    else:
        _check_opt(out, n_out, odt, "out")
    check(lib.sengine_amd_fused_sparse_conv_bn_add_neuron(
        p.ref, _ptr(data), _ptr(values), _ptr(meta), _ptr(state), _ptr(bn_scale), _ptr(bn_bias), _ptr(residual),
        _ptr(real_out), _ptr(out), _stream(dev)), "fused_sparse_conv_bn_add_neuron")
    return real_out, out


def real_conv_bn(s: ConvSpec, x: torch.Tensor, weight: torch.Tensor, bn_scale: torch.Tensor, bn_bias: torch.Tensor,
                 in_T: Optional[int] = None, out: Optional[torch.Tensor] = None,
                 layout: int = WLAYOUT_OIHW) -> torch.Tensor:
    """MS-ResNet shortcut: fp32 1x1 conv (stride s.stride) + folded BN on the real-valued
    NHWC input x (in_T*s.B, H, W, C_in) -> fp32 NHWC (s.T*s.B, OH, OW, C_out).  in_T = 1
    (one timestep of input, e.g. the stem output) stores every output value s.T times;
    default in_T = s.T.  weight: OIHW (C_out, C_in, 1, 1) or HWIO (1, 1, C_in, C_out)."""
    lib = _lib.load()
    in_T = s.T if in_T is None else in_T
    for t, n in ((x, "x"), (weight, "weight"), (bn_scale, "bn_scale"), (bn_bias, "bn_bias")):
        _require_cuda(t, n)
    _require_numel(x, in_T * s.B * s.H * s.W * s.C_in, torch.float32, "x")
    _require_numel(weight, s.C_out * s.C_in, torch.float32, "weight")
    _require_numel(bn_scale, s.C_out, torch.float32, "bn_scale")
    _require_numel(bn_bias, s.C_out, torch.float32, "bn_bias")
    OH, OW = (s.H - 1) // s.stride + 1, (s.W - 1) // s.stride + 1
    if out is None:
        out = torch.empty(s.T * s.B, OH, OW, s.C_out, dtype=torch.float32, device=x.device)
    else:
        _require_cuda(out, "out")
        _require_numel(out, s.T * s.B * OH * OW * s.C_out, torch.float32, "out")
    d = make_desc(s)
    check(lib.sengine_amd_real_conv_bn(ctypes.byref(d), _ptr(x), int(in_T), _ptr(weight), int(layout),
                                       _ptr(bn_scale), _ptr(bn_bias), _ptr(out), _stream(x.device)), "real_conv_bn")
    return out


def attention_needs_kv(T: int, B: int, N: int, C: int, heads: int, workspace: bool = False) -> bool:
    """Whether spiking_self_attention runs as two kernels with K^T V in a workspace between them
    (else one kernel keeps it in LDS): of a call without `kv`, or with one (workspace=True)."""
    return bool(_lib.load().sengine_amd_ssa_attention_needs_kv(T, B, N, C, heads, int(workspace)))


def spiking_self_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, T: int, B: int, N: int, C: int,
                           heads: int, scale: float = 0.125, neuron: str = "lif", tau: float = 2.0,
                           v_threshold: float = 0.5, v_reset: Optional[float] = 0.0,
                           kv: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Spikformer SSA on spike bits: q, k, v int32 (T*B, N, C/32) -> the attention neuron's
    spikes over T of (Q K^T * scale) V per head, int32 (T*B, N, C/32).  kv: optional
    workspace int32 (T*B, heads, d, d) (K^T V per head)."""
    lib = _lib.load()
    n_bits = T * B * N * C // 32
    for t, name in ((q, "q"), (k, "k"), (v, "v")):
        _check_req(t, n_bits, torch.int32, name)
    d = C // heads if heads else 0
    if kv is not None:
        _check_req(kv, T * B * heads * d * d, torch.int32, "kv")
    elif attention_needs_kv(T, B, N, C, heads):
        kv = torch.empty((T * B, heads, d, d), dtype=torch.int32, device=q.device)
    if out is None:
        out = torch.empty((T * B, N, C // 32), dtype=torch.int32, device=q.device)
    else:
        _check_req(out, n_bits, torch.int32, "out")
    hard = v_reset is not None
    check(lib.sengine_amd_ssa_attention(T, B, N, C, heads, float(scale), neuron_code(neuron), int(hard), float(tau),
                                        float(v_threshold), float(v_reset if hard else 0.0), q.data_ptr(),
                                        k.data_ptr(), v.data_ptr(), _ptr(kv), out.data_ptr(), _stream(q.device)),
          "ssa_attention")
    return out


def stem_conv_bn(s: ConvSpec, x: torch.Tensor, weight: torch.Tensor, bn_scale: torch.Tensor, bn_bias: torch.Tensor,
                 out: Optional[torch.Tensor] = None, layout: int = WLAYOUT_OIHW) -> torch.Tensor:
    """Dense fp32 conv + folded BN on NCHW images (s.B images; s.T ignored) -> NHWC fp32.
    weight: OIHW, or HWIO (KH, KW, C_in, C_out) with layout=WLAYOUT_HWIO (coalesced reads)."""
    lib = _lib.load()
    for t, n in ((x, "x"), (weight, "weight"), (bn_scale, "bn_scale"), (bn_bias, "bn_bias")):
        _require_cuda(t, n)
    _require_numel(x, s.B * s.C_in * s.H * s.W, torch.float32, "x")
    _require_numel(weight, s.C_out * s.C_in * s.KH * s.KW, torch.float32, "weight")
    _require_numel(bn_scale, s.C_out, torch.float32, "bn_scale")
    _require_numel(bn_bias, s.C_out, torch.float32, "bn_bias")
    OH = (s.H + 2 * s.padding - s.KH) // s.stride + 1
    OW = (s.W + 2 * s.padding - s.KW) // s.stride + 1
    if out is None:
        out = torch.empty(s.B, OH, OW, s.C_out, dtype=torch.float32, device=x.device)
    else:
        _require_cuda(out, "out")
        _require_numel(out, s.B * OH * OW * s.C_out, torch.float32, "out")
    d = make_desc(s)
    check(lib.sengine_amd_stem_conv_bn(ctypes.byref(d), _ptr(x), _ptr(weight), int(layout), _ptr(bn_scale),
                                       _ptr(bn_bias), _ptr(out), _stream(x.device)), "stem_conv_bn")
    return out


def stem_conv_bn_lif_pool(s: ConvSpec, x: torch.Tensor, weight_hwio: torch.Tensor, bn_scale: torch.Tensor,
                          bn_bias: torch.Tensor, pool_k: int = 3, pool_stride: int = 2, pool_pad: int = 1,
                          pooled: Optional[torch.Tensor] = None, spikes: Optional[torch.Tensor] = None):
    """Stem conv + folded BN, the neuron of `s` over the output repeated s.T times, and
    MaxPool2d(pool_k, pool_stride, pool_pad) of the spikes, in one launch.  Returns
    (pooled, spikes): int32 spike-bit tensors (s.T*s.B, POH, POW, C_out/32) and, if a
    `spikes` buffer is given, the stem spikes (s.T*s.B, OH, OW, C_out/32) (else None)."""
    lib = _lib.load()
    for t, n in ((x, "x"), (weight_hwio, "weight_hwio"), (bn_scale, "bn_scale"), (bn_bias, "bn_bias")):
        _require_cuda(t, n)
    _require_numel(x, s.B * s.C_in * s.H * s.W, torch.float32, "x")
    _require_numel(weight_hwio, s.C_out * s.C_in * s.KH * s.KW, torch.float32, "weight_hwio")
    _require_numel(bn_scale, s.C_out, torch.float32, "bn_scale")
    _require_numel(bn_bias, s.C_out, torch.float32, "bn_bias")
    OH = (s.H + 2 * s.padding - s.KH) // s.stride + 1
    OW = (s.W + 2 * s.padding - s.KW) // s.stride + 1
    POH = (OH + 2 * pool_pad - pool_k) // pool_stride + 1
    POW = (OW + 2 * pool_pad - pool_k) // pool_stride + 1
    if pooled is None:
        pooled = torch.empty(s.T * s.B, POH, POW, s.C_out // 32, dtype=torch.int32, device=x.device)
    else:
        _require_cuda(pooled, "pooled")
        _require_numel(pooled, s.T * s.B * POH * POW * s.C_out // 32, torch.int32, "pooled")
    if spikes is not None:
        _require_cuda(spikes, "spikes")
        _require_numel(spikes, s.T * s.B * OH * OW * s.C_out // 32, torch.int32, "spikes")
    d = make_desc(s)
    check(lib.sengine_amd_stem_conv_bn_lif_pool(ctypes.byref(d), _ptr(x), _ptr(weight_hwio), _ptr(bn_scale),
                                                _ptr(bn_bias), int(pool_k), int(pool_stride), int(pool_pad),
                                                _ptr(spikes) if spikes is not None else None, _ptr(pooled),
                                                _stream(x.device)), "stem_conv_bn_lif_pool")
    return pooled, spikes


def stem_conv_bn_neuron(s: ConvSpec, x: torch.Tensor, weight_hwio: torch.Tensor, bn_scale: torch.Tensor,
                        bn_bias: torch.Tensor, out: Optional[torch.Tensor] = None, spikes: Optional[torch.Tensor] = None,
                        want_out: bool = True):
    """Stem conv + folded BN (NHWC fp32 `out`, skipped when want_out is False and no `out`
    is given) and the neuron of `s` over that output repeated s.T times (spike bits int32
    (s.T*s.B, OH, OW, C_out/32), the layout of multistep_neuron_repeat on `out`), in one
    launch.  Returns (out or None, spikes)."""
    lib = _lib.load()
    _check_req(x, s.B * s.C_in * s.H * s.W, torch.float32, "x")
    _check_req(weight_hwio, s.C_out * s.C_in * s.KH * s.KW, torch.float32, "weight_hwio")
    _check_req(bn_scale, s.C_out, torch.float32, "bn_scale")
    _check_req(bn_bias, s.C_out, torch.float32, "bn_bias")
    OH = (s.H + 2 * s.padding - s.KH) // s.stride + 1
    OW = (s.W + 2 * s.padding - s.KW) // s.stride + 1
    if out is None and want_out:
        out = torch.empty((s.B, OH, OW, s.C_out), dtype=torch.float32, device=x.device)
    else:
        _check_opt(out, s.B * OH * OW * s.C_out, torch.float32, "out")
    if spikes is None:
        spikes = torch.empty((s.T * s.B, OH, OW, s.C_out // 32), dtype=torch.int32, device=x.device)
    else:
        _check_req(spikes, s.T * s.B * OH * OW * s.C_out // 32, torch.int32, "spikes")
    check(lib.sengine_amd_stem_conv_bn_neuron(_ref(s), x.data_ptr(), weight_hwio.data_ptr(), bn_scale.data_ptr(),
                                              bn_bias.data_ptr(), _ptr(out), spikes.data_ptr(), _stream(x.device)),
          "stem_conv_bn_neuron")
    return out, spikes


def multistep_neuron_repeat(x: torch.Tensor, T: int, neuron: str = "lif", tau: float = 2.0, v_threshold: float = 1.0,
                            v_reset: Optional[float] = 0.0, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Neuron over T steps of the same input x (fp32, n % 32 == 0): spike bits int32 (T, n/32)."""
    lib = _lib.load()
    _require_cuda(x, "x")
    if x.dtype != torch.float32:
        raise SEngineError("multistep_neuron_repeat: x must be fp32")
    n = x.numel()
    if out is None:
        out = torch.empty(T, n // 32, dtype=torch.int32, device=x.device)
    else:
        _require_cuda(out, "out")
        _require_numel(out, T * n // 32, torch.int32, "out")
    hard = v_reset is not None
    check(lib.sengine_amd_multistep_neuron_repeat(int(T), int(n), neuron_code(neuron),
                                                  int(hard), float(tau), float(v_threshold),
                                                  float(v_reset if hard else 0.0), _ptr(x), _ptr(out),
                                                  _stream(x.device)), "multistep_neuron_repeat")
    return out


def maxpool_spikes(x: torch.Tensor, NT: int, H: int, W: int, C: int, k: int = 3, stride: int = 2, pad: int = 1,
                   out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Max-pool spike bits (NT, H, W, C/32 words) -> (NT, OH, OW, C/32)."""
    lib = _lib.load()
    _require_cuda(x, "x")
    _require_numel(x, NT * H * W * C // 32, torch.int32, "x")
    OH, OW = (H + 2 * pad - k) // stride + 1, (W + 2 * pad - k) // stride + 1
    if out is None:
        out = torch.empty(NT, OH, OW, C // 32, dtype=torch.int32, device=x.device)
    else:
        _require_cuda(out, "out")
        _require_numel(out, NT * OH * OW * C // 32, torch.int32, "out")
    check(lib.sengine_amd_maxpool_spikes(NT, H, W, C, k, stride, pad, _ptr(x), _ptr(out), _stream(x.device)),
          "maxpool_spikes")
    return out


HEAD_WS_SPLIT = 64  # summing workgroups per image of sengine_amd_sew_head_ws (workspace B * 64 * C)


def sew_head(x: torch.Tensor, T: int, B: int, HW: int, C: int, planes: int, fc_weight: torch.Tensor,
             fc_bias: torch.Tensor, out: Optional[torch.Tensor] = None,
             workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Average pool + mean over T + Linear on `planes`-plane integer activations (planes = 0:
    integer-valued fp16 (T*B, HW, C)) -> (B, N_out) fp32.  fc_weight: (N_out, C) contiguous,
    nn.Linear layout.  With `workspace` (int32, at least B * 64 * C elements) an fp16 stream's
    sums are split over many workgroups per image (sengine_amd_sew_head_ws)."""
    lib = _lib.load()
    for t, n in ((x, "x"), (fc_weight, "fc_weight"), (fc_bias, "fc_bias")):
        _require_cuda(t, n)
    if planes == 0:
        _require_numel(x, T * B * HW * C, torch.float16, "x")
    else:
        _require_numel(x, T * B * HW * planes * C // 32, torch.int32, "x")
    N_out = fc_weight.shape[0]
    _require_numel(fc_weight, N_out * C, torch.float32, "fc_weight")
    _require_numel(fc_bias, N_out, torch.float32, "fc_bias")
    if out is None:
        out = torch.empty(B, N_out, dtype=torch.float32, device=x.device)
    else:
        _require_cuda(out, "out")
        _require_numel(out, B * N_out, torch.float32, "out")
    if workspace is not None:
        _require_cuda(workspace, "workspace")
        if workspace.dtype != torch.int32 or workspace.numel() < B * HEAD_WS_SPLIT * C:
            raise SEngineError(f"workspace: need >= {B * HEAD_WS_SPLIT * C} int32 elements")
        check(lib.sengine_amd_sew_head_ws(T, B, HW, C, planes, _ptr(x), _ptr(fc_weight), _ptr(fc_bias), N_out,
                                          _ptr(out), _ptr(workspace), workspace.numel(), _stream(x.device)),
              "sew_head_ws")
        return out
    check(lib.sengine_amd_sew_head(T, B, HW, C, planes, _ptr(x), _ptr(fc_weight), _ptr(fc_bias), N_out, _ptr(out),
                                   _stream(x.device)), "sew_head")
    return out


def dense_conv_bn(s: ConvSpec, data: torch.Tensor, values: torch.Tensor, bn_scale: torch.Tensor,
                  bn_bias: torch.Tensor, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Dense Conv + folded BN -> fp32 (T*B, OH, OW, C_out)."""
    lib = _lib.load()
    p = _plan(s)
    vb = p.dense_blob()
    _require_cuda(values, "values")
    dt, n_in = p.data(s)
    _check_req(data, n_in, dt, "data")
    if values.nbytes != vb:
        raise SEngineError("dense_conv_bn: weight blob does not match the descriptor")
    _check_req(bn_scale, s.C_out, torch.float32, "bn_scale")
    _check_req(bn_bias, s.C_out, torch.float32, "bn_bias")
    if out is None:
        out = torch.empty((s.T * s.B, p.OH, p.OW, s.C_out), dtype=torch.float32, device=data.device)
    else:
        _check_opt(out, s.T * p.M * s.C_out, torch.float32, "out")
    check(lib.sengine_amd_dense_conv_bn(p.ref, _ptr(data), _ptr(values), _ptr(bn_scale), _ptr(bn_bias), _ptr(out),
                                        _stream(data.device)), "dense_conv_bn")
    return out


def multistep_neuron(x: torch.Tensor, T: int, neuron: str = "lif", tau: float = 2.0, v_threshold: float = 1.0,
                     v_reset: Optional[float] = 0.0, state: Optional[torch.Tensor] = None, out_enc: int = ENC_BITS,
                     h_trace: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Standalone multi-step LIF/IF over T on x (T, ...) fp32 (n = x.numel()/T per step).
    v_reset=None selects soft reset (models/neurons.py:135-137).  Returns spikes as bits
    int32 (T, n/32) or fp16 (T, n)."""
    lib = _lib.load()
    _require_cuda(x, "x")
    if x.dtype != torch.float32 or x.numel() % T:
        raise SEngineError("multistep_neuron: x must be fp32 with T * n elements")
    n = x.numel() // T
    _check_opt(state, n, torch.float32, "state")
    _check_opt(h_trace, T * n, torch.float32, "h_trace")
    odt, n_out = _enc_numel(out_enc, T * n)
    if out is None:
        out = torch.empty(n_out, dtype=odt, device=x.device)
    else:
        _check_req(out, n_out, odt, "out")
    hard = v_reset is not None
    check(lib.sengine_amd_multistep_neuron(T, n, neuron_code(neuron), int(hard), float(tau),
                                           float(v_threshold), float(v_reset if hard else 0.0), _ptr(x), _ptr(state),
                                           out_enc, _ptr(out), _ptr(h_trace), _stream(x.device)), "multistep_neuron")
    return out


# ------------------------------------------------------------------ token operators

_TOKEN_TYPES = {torch.float16: ENC_F16, torch.bfloat16: ENC_BF16, torch.float32: ENC_F32,
                torch.float8_e4m3fn: ENC_E4M3}


_NOT_RECORDED = ("the token operators cannot be recorded by a tracer, which would see their outputs' allocation only "
                 "(capture a HIP graph instead)")
_dispatch_modes = torch._C._len_torch_dispatch_stack


def _token_modes(*args):
    """What a call refuses that its arguments' layouts do not show: tangents of forward-mode differentiation (there is no
    rule for them, and no_grad does not turn them off), and a recording by torch.fx."""
    for t in args:
        if isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None:
            raise SEngineError("an input has a tangent: the token operators are inference only "
                               "(call them outside of forward_ad.dual_level())")
    if torch._C._get_dispatch_mode(torch._C._TorchDispatchModeKey.PROXY) is not None:
        raise SEngineError(_NOT_RECORDED)


def _type_code(t: torch.Tensor, allowed, name: str) -> int:
    if t.dtype not in allowed:
        raise SEngineError(f"{name}: expected dtype {' or '.join(str(d) for d in allowed)}, got {t.dtype}")
    return _TOKEN_TYPES[t.dtype]


def _token_input(t, name: str, device=None):
    """A tensor that a token operator reads: on the device, and not one that asks for a gradient
    (these operators have no backward; it is refused rather than cut off)."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if torch.jit.is_tracing():  # shapes are tensors then, so that no call is found among the remembered ones
        raise SEngineError(_NOT_RECORDED)
    if not t.is_cuda:
        raise SEngineError(f"{name} must be on a HIP device (got {t.device})")
    if device is not None and t.device != device:
        raise SEngineError(f"{name} is on {t.device}, the others on {device}")
    if t.requires_grad and torch.is_grad_enabled():
        raise SEngineError(f"{name} requires a gradient: the token operators are inference only "
                           "(call them under torch.no_grad())")


def _token_number(x, name: str) -> float:
    """eps or scale as the number it is at the call (a tensor's value may be another one at the next), to 32 bits."""
    if isinstance(x, torch.Tensor) and x.requires_grad and torch.is_grad_enabled():
        raise SEngineError(f"{name} requires a gradient: the token operators are inference only "
                           "(call them under torch.no_grad())")
    return ctypes.c_float(x).value


def _token_sizes(what: str, *sizes):
    """Sizes that the descriptors hold in 32 bits; ctypes would cut them without a word."""
    if max(sizes) >= 2**31:
        raise SEngineError(f"{what} must be under 2**31, got {', '.join(map(str, sizes))}")


def _token_rows(t: torch.Tensor, name: str):
    """(rows, row stride in elements) of (..., width), whose rows must lie evenly spaced."""
    if t.is_contiguous():
        return (t.numel() // t.shape[-1] if t.shape[-1] else math.prod(t.shape[:-1])), t.shape[-1]
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        raise SEngineError(f"{name}: the values of a row must lie side by side")
    dims = [(n, st) for n, st in zip(t.shape[:-1], t.stride()[:-1]) if n != 1]
    for (_, outer), (n, inner) in zip(dims, dims[1:]):
        if outer != n * inner:
            raise SEngineError(f"{name}: the rows must be evenly spaced (shape {tuple(t.shape)}, "
                               f"strides {t.stride()})")
    return math.prod(t.shape[:-1]), dims[-1][1] if dims else t.shape[-1]


def _token_vector(t, n: int, name: str, device):
    _token_input(t, name, device)
    if t.numel() != n or not t.is_contiguous():
        raise SEngineError(f"{name}: expected {n} contiguous elements, got shape {tuple(t.shape)}")


def _token_out(t, shape, dtype, name: str, device):
    """An output given by the caller; returns its row stride."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if t.device != device:
        raise SEngineError(f"{name} is on {t.device}, the input on {device}")
    if t.dtype != dtype or tuple(t.shape) != tuple(shape):
        raise SEngineError(f"{name}: expected {dtype} {tuple(shape)}, got {t.dtype} {tuple(t.shape)}")
    if t.requires_grad and torch.is_grad_enabled():
        raise SEngineError(f"{name} requires a gradient: the token operators are inference only")
    return _token_rows(t, name)[1]


# What a call's checks come to depends on its tensors' types, shapes, strides and devices only; it is kept under them,
# so that the calls of a decoding loop do not pay for the checks again (they take longer than a small kernel).
_TOKEN_PLANS: dict = {}


def _remember(key, plan):
    if key is not None:
        if len(_TOKEN_PLANS) >= 4096:
            _TOKEN_PLANS.clear()
        _TOKEN_PLANS[key] = plan
    return plan


def _layout(t):
    return None if t is None else (t.dtype, t.shape, t.stride(), t.device)


_current_device = getattr(torch._C, "_cuda_getDevice", lambda: 0)  # absent in CPU-only builds


def _launch(entry, device: torch.device, what: str, *args):
    """Calls an entry with its device as the current one: the default stream's handle is the same for every device."""
    if device.index == _current_device():
        check(entry(*args, _stream(device)), what)
    else:
        with torch.cuda.device(device):
            check(entry(*args, _stream(device)), what)


def _rms_norm_plan(key, x, weight, residual, eps, out_dtype, out, stream_out, scale):
    """(descriptor, output's type, whether that is e4m3, rows' shape, device, whether x is dense) of a checked call."""
    _token_input(x, "x")
    dev, code = x.device, _type_code(x, (torch.float16, torch.bfloat16, torch.float32), "x")
    if x.dim() == 0:
        raise SEngineError("x: expected (..., D)")
    shape, D = x.shape, x.shape[-1]
    _token_sizes("rms_norm: D", D)
    rows, xs = _token_rows(x, "x")
    rs = ws = 0
    if residual is not None:
        _token_input(residual, "residual", dev)
        if residual.shape != shape or residual.dtype != x.dtype:
            raise SEngineError(f"residual: expected {x.dtype} {tuple(shape)}, got {residual.dtype} "
                               f"{tuple(residual.shape)}")
        rs = _token_rows(residual, "residual")[1]
    elif stream_out is not None:
        raise SEngineError("stream_out: there is no residual to add")
    if weight is not None:
        _token_vector(weight, D, "weight", dev)
        ws = _type_code(weight, (x.dtype, torch.float32), "weight")
    eight = out_dtype is torch.float8_e4m3fn
    if out_dtype is None:
        out_dtype = x.dtype
    elif out_dtype is not x.dtype and not eight:
        raise SEngineError(f"out_dtype: expected {x.dtype} or torch.float8_e4m3fn, got {out_dtype}")
    os_ = D if out is None else _token_out(out, shape, out_dtype, "out", dev)
    ss = D if stream_out is None else _token_out(stream_out, shape, x.dtype, "stream_out", dev)
    if scale is not None:
        if not eight:
            raise SEngineError("scale goes with out_dtype=torch.float8_e4m3fn")
        _token_vector(scale, rows, "scale", dev)
        _type_code(scale, (torch.float32,), "scale")
    desc = ctypes.byref(RmsNormDesc(rows, xs, rs, os_, ss, D, code, ws, _TOKEN_TYPES[out_dtype], eps))
    return _remember(key, (desc, out_dtype, eight, shape, dev, x.is_contiguous()))


def rms_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, residual: Optional[torch.Tensor] = None,
             eps: float = 1e-6, out_dtype: Optional[torch.dtype] = None, out: Optional[torch.Tensor] = None,
             stream_out: Optional[torch.Tensor] = None, scale: Optional[torch.Tensor] = None):
    """Root-mean-square norm of rows x (..., D) with the residual's addition: s = x + residual,
    y = s / sqrt(mean(s^2) + eps) * weight, in fp32, y formed from the unrounded s.

    x is fp16, bf16 or fp32; residual and stream have its shape and type; weight (D,) its type or
    fp32.  Returns (y, stream) with y in x's type, or with out_dtype=torch.float8_e4m3fn
    (y, stream, scale): y's codes and one fp32 scale a row (shape x.shape[:-1]), y ~ codes * scale, which is
    max|y| / 448, at least 2**-126 and 1 for a row of zeros.
    stream is s rounded to x's type, None without a residual.  `out`, `stream_out` (which may be
    `residual`, updated in place) and `scale` take the results where given."""
    if _dispatch_modes() or forward_ad._current_level >= 0:
        _token_modes(x, weight, residual, eps)
    if type(eps) is not float:
        eps = _token_number(eps, "eps")
    key = None
    if out is None and stream_out is None and scale is None:
        try:
            key = ("norm", x.dtype, x.shape, x.stride(), x.device, eps, out_dtype, _layout(weight), _layout(residual))
        except AttributeError:
            pass  # not a tensor: the checks say so
    plan = _TOKEN_PLANS.get(key)
    if plan is None or (torch.is_grad_enabled() and (
            x.requires_grad or (weight is not None and weight.requires_grad)
            or (residual is not None and residual.requires_grad))):
        plan = _rms_norm_plan(key, x, weight, residual, eps, out_dtype, out, stream_out, scale)
    desc, out_dtype, eight, shape, dev, dense = plan
    if out is None:
        out = torch.empty(shape, dtype=out_dtype, device=dev) if eight or not dense else torch.empty_like(x)
    if residual is not None and stream_out is None:
        stream_out = torch.empty_like(x) if dense else torch.empty(shape, dtype=x.dtype, device=dev)
    if eight and scale is None:
        scale = torch.empty(shape[:-1], dtype=torch.float32, device=dev)
    _launch(_lib.load().sengine_amd_rms_norm, dev, "rms_norm", desc, x.data_ptr(), _ptr(residual), _ptr(weight),
            out.data_ptr(), _ptr(stream_out), _ptr(scale))
    return (out, stream_out, scale) if eight else (out, stream_out)


def _linear_plan(key, x, weight, bias, activation, residual, x_scale, weight_scale, out_dtype, out):
    """(descriptor, bytes of scratch memory, output's shape and type, device) of a checked call."""
    _token_input(x, "x")
    dev = x.device
    code = _type_code(x, (torch.float16, torch.bfloat16, torch.float8_e4m3fn), "x")
    _token_input(weight, "weight", dev)
    if x.dim() == 0 or weight.dim() != 2 or weight.dtype != x.dtype or weight.shape[1] != x.shape[-1]:
        raise SEngineError(f"weight: expected {x.dtype} (N, K) for x {tuple(x.shape)}, got {weight.dtype} "
                           f"{tuple(weight.shape)}")
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {sorted(ACTIVATIONS)}, got {activation!r}")
    N, K = weight.shape
    _token_sizes("linear: N and K", N, K)
    M, xs = _token_rows(x, "x")
    wst = _token_rows(weight, "weight")[1]
    eight = code == ENC_E4M3
    if out_dtype is None:
        out_dtype = torch.bfloat16 if eight else x.dtype
    ocode = _TOKEN_TYPES.get(out_dtype, ENC_E4M3)
    if ocode == ENC_E4M3:
        raise SEngineError(f"out_dtype: expected float16, bfloat16 or float32, got {out_dtype}")
    for t, n, name in ((x_scale, M, "x_scale"), (weight_scale, N, "weight_scale")):
        if t is not None:
            if not eight:
                raise SEngineError(f"{name} goes with float8_e4m3fn operands")
            _token_vector(t, n, name, dev)
            _type_code(t, (torch.float32,), name)
    bcode = 0
    if bias is not None:
        _token_vector(bias, N, "bias", dev)
        bcode = _type_code(bias, (torch.float16, torch.bfloat16, torch.float32), "bias")
    shape = (*x.shape[:-1], N)
    rs = 0
    if residual is not None:
        _token_input(residual, "residual", dev)
        if residual.shape != shape or residual.dtype != out_dtype:
            raise SEngineError(f"residual: expected {out_dtype} {shape}, got {residual.dtype} "
                               f"{tuple(residual.shape)}")
        rs = _token_rows(residual, "residual")[1]
    os_ = N if out is None else _token_out(out, shape, out_dtype, "out", dev)
    desc = ctypes.byref(LinearDesc(M, xs, wst, rs, os_, N, K, code, ocode, bcode, ACTIVATIONS[activation]))
    size = ctypes.c_size_t()
    check(_lib.load().sengine_amd_linear_workspace(desc, ctypes.byref(size)), "linear")
    return _remember(key, (desc, size.value, shape, out_dtype, dev))


def linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, activation: str = "none",
           residual: Optional[torch.Tensor] = None, x_scale: Optional[torch.Tensor] = None,
           weight_scale: Optional[torch.Tensor] = None, out_dtype: Optional[torch.dtype] = None,
           out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """act(x weight^T + bias) + residual of token rows x (..., K) with weight (N, K), nn.Linear's
    layout; activation 'none' | 'relu' | 'gelu' (by the error function) | 'gelu_tanh' | 'silu'.

    x and weight are both fp16, both bf16, or both float8_e4m3fn with fp32 scales of x's rows
    (x_scale, as rms_norm returns it) and of weight's rows (weight_scale, (N,)).  The sums and what
    follows them are fp32; the 8-bit matrix instructions that make 16-bit results of e4m3 operands are
    off by up to 2**-12 of the sum of the products' magnitudes (a tenth of an fp16 rounding, but more
    of a sum that cancels), and an fp32 result takes the 16-bit instructions instead, at half the
    rate, with sums of 32 bits.  The result is rounded once to out_dtype (fp16, bf16 or fp32; x's
    type, for e4m3 bf16, by default).  residual (..., N) has out_dtype, bias (N,) fp16, bf16 or fp32;
    `out` may be `residual` but must share no memory with x or weight.  A long reduction with few
    results is computed in parts through scratch memory of torch's allocator, the parts added in a
    fixed order."""
    if _dispatch_modes() or forward_ad._current_level >= 0:
        _token_modes(x, weight, bias, residual, x_scale, weight_scale)
    key = None
    if out is None:
        try:
            key = ("linear", x.dtype, x.shape, x.stride(), x.device, weight.dtype, weight.shape, weight.stride(),
                   weight.device, activation, out_dtype, _layout(bias), _layout(residual), _layout(x_scale),
                   _layout(weight_scale))
        except AttributeError:
            pass  # not a tensor: the checks say so
    plan = _TOKEN_PLANS.get(key)
    if plan is None or (torch.is_grad_enabled() and (
            x.requires_grad or weight.requires_grad
            or any(t is not None and t.requires_grad for t in (bias, residual, x_scale, weight_scale)))):
        plan = _linear_plan(key, x, weight, bias, activation, residual, x_scale, weight_scale, out_dtype, out)
    desc, size, shape, out_dtype, dev = plan
    if out is None:
        out = torch.empty(shape, dtype=out_dtype, device=dev)
    ws = torch.empty(size, dtype=torch.uint8, device=dev) if size else None
    _launch(_lib.load().sengine_amd_linear_ws, dev, "linear", desc, x.data_ptr(), weight.data_ptr(), _ptr(x_scale),
            _ptr(weight_scale), _ptr(bias), _ptr(residual), out.data_ptr(), _ptr(ws), size)
    return out


def _cross_plan(key, q, k, v, scale, key_lengths, key_mask, out):
    """(descriptor, bytes of scratch memory, device) of a checked call."""
    _token_input(q, "q")
    dev, code = q.device, _type_code(q, (torch.float16, torch.bfloat16), "q")
    for t, name in ((k, "k"), (v, "v")):
        _token_input(t, name, dev)
        if t.dtype != q.dtype:
            raise SEngineError(f"{name}: expected {q.dtype}, got {t.dtype}")
    if q.dim() != 4 or k.dim() != 4 or v.shape != k.shape or k.shape[0] != q.shape[0] or k.shape[3] != q.shape[3]:
        raise SEngineError(f"cross_attention: expected q (B, Lq, Hq, d) and k, v (B, Lk, Hkv, d), got "
                           f"{tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    B, Lq, Hq, d = q.shape
    Lk, Hkv = k.shape[1], k.shape[2]
    _token_sizes("cross_attention: B, Lq, Lk, heads and d", B, Lq, Lk, Hq, Hkv, d)
    if out is not None:
        if not isinstance(out, torch.Tensor):
            raise TypeError("out must be a torch.Tensor")
        if out.device != dev or out.dtype != q.dtype or out.shape != q.shape:
            raise SEngineError(f"out: expected {q.dtype} {tuple(q.shape)} on {dev}, got {out.dtype} "
                               f"{tuple(out.shape)} on {out.device}")
        if out.requires_grad and torch.is_grad_enabled():
            raise SEngineError("out requires a gradient: the token operators are inference only")
    st = [t.stride() for t in (q, k, v)]
    st.append(out.stride() if out is not None else (Lq * Hq * d, Hq * d, d, 1))
    for t, s, name in zip((q, k, v, q if out is None else out), st, ("q", "k", "v", "out")):
        if t.numel() and ((s[3] != 1 and d > 1) or any(n > 1 and x % 8 for n, x in zip(t.shape, s[:3]))):
            raise SEngineError(f"{name}: rows of d values must be contiguous and begin at multiples of 16 bytes "
                               f"(strides {s})")
    if key_lengths is not None:
        _token_vector(key_lengths, B, "key_lengths", dev)
        if key_lengths.dtype != torch.int32:
            raise SEngineError(f"key_lengths: expected dtype torch.int32, got {key_lengths.dtype}")
    ms = 0
    if key_mask is not None:
        _token_input(key_mask, "key_mask", dev)
        if key_mask.dtype != torch.bool or key_mask.shape != (B, Lk) or (Lk > 1 and key_mask.stride(1) != 1):
            raise SEngineError(f"key_mask: expected torch.bool ({B}, {Lk}) with contiguous rows, got "
                               f"{key_mask.dtype} {tuple(key_mask.shape)}")
        ms = key_mask.stride(0)
    s3 = ctypes.c_int64 * 3
    # a stride over a single element is never taken: 0 keeps it from looking unaligned
    st = [s3(*(x if n > 1 else 0 for n, x in zip(t.shape[:3], s))) for t, s in zip((q, k, v, q), st)]
    desc = ctypes.byref(CrossDesc(*st, ms, B, Lq, Lk, Hq, Hkv, d, code, 1.0 / math.sqrt(d) if scale is None else scale))
    size = ctypes.c_size_t()
    check(_lib.load().sengine_amd_cross_attention_workspace(desc, ctypes.byref(size)), "cross_attention")
    return _remember(key, (desc, size.value, dev))


def cross_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: Optional[float] = None,
                    key_lengths: Optional[torch.Tensor] = None, key_mask: Optional[torch.Tensor] = None,
                    out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of q (B, Lq, Hq, d) to an encoder's states k, v (B, Lk, Hkv, d), Hq a multiple of
    Hkv (query head h reads key head h // (Hq // Hkv)), d a multiple of 8 up to 128; fp16 or bf16;
    scale 1 / sqrt(d) by default.  Returns (B, Lq, Hq, d) in q's type.

    key_lengths (B,) int32: the keys of each sequence that count (clamped to 0..Lk); key_mask
    (B, Lk) bool: True where a key counts.  A query with no key that counts gets zeros; what lies
    in the others is never used.  Any strides whose rows of d values are contiguous and begin at
    multiples of 16 bytes; k and v expanded over the batch (one encoder pass, many queries) are read
    as they are.  Scores, their maximum and sums are fp32; the weights are rounded to q's type for
    the product with v, fp16 ones down to 2**-31 of the largest.  `out` may be q but must share no
    memory with k or v.  Few queries of many keys are computed in parts of the keys through scratch
    memory of torch's allocator, the parts joined in a fixed order."""
    if _dispatch_modes() or forward_ad._current_level >= 0:
        _token_modes(q, k, v, scale)
    if scale is not None and type(scale) is not float:
        scale = _token_number(scale, "scale")
    key = None
    if out is None:
        try:
            key = ("cross", q.dtype, q.shape, q.stride(), q.device, k.dtype, k.shape, k.stride(), k.device, v.dtype,
                   v.shape, v.stride(), v.device, scale, _layout(key_lengths), _layout(key_mask))
        except AttributeError:
            pass  # not a tensor: the checks say so
    plan = _TOKEN_PLANS.get(key)
    if plan is None or (torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad)):
        plan = _cross_plan(key, q, k, v, scale, key_lengths, key_mask, out)
    desc, size, dev = plan
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=dev)
    qp, kp, vp, op = q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr()
    if (qp | kp | vp | op) & 15:
        for p, t, name in ((qp, q, "q"), (kp, k, "k"), (vp, v, "v"), (op, out, "out")):
            if p & 15 and t.numel():
                raise SEngineError(f"{name}: must begin at a multiple of 16 bytes")
    ws = torch.empty(size, dtype=torch.uint8, device=dev) if size else None
    _launch(_lib.load().sengine_amd_cross_attention_ws, dev, "cross_attention", desc, qp, kp, vp, _ptr(key_lengths),
            _ptr(key_mask), op, _ptr(ws), size)
    return out


def _heads_out(t, shape, dtype, name: str, device):
    """An output (B, L, heads, d) given by the caller: any strides, the values of a head side by side."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if t.device != device or t.dtype != dtype or t.shape != shape:
        raise SEngineError(f"{name}: expected {dtype} {tuple(shape)} on {device}, got {t.dtype} {tuple(t.shape)} on "
                           f"{t.device}")
    if t.requires_grad and torch.is_grad_enabled():
        raise SEngineError(f"{name} requires a gradient: the token operators are inference only")


def _head_strides(t, name: str):
    """Strides per (batch, token, head) of (B, L, heads, d), whose heads' values must lie side by side."""
    s = t.stride()
    if t.numel() and t.shape[3] > 1 and s[3] != 1:
        raise SEngineError(f"{name}: the values of a head must lie side by side (strides {s})")
    # a stride over a single element is never taken: 0 keeps it from looking unaligned
    return (ctypes.c_int64 * 3)(*(x if n > 1 else 0 for n, x in zip(t.shape[:3], s)))


def _rotary_plan(key, q, k, positions, frequencies, sections, interleaved, out_q, out_k):
    """(descriptor, device) of a checked call."""
    _token_input(q, "q")
    dev, code = q.device, _type_code(q, (torch.float16, torch.bfloat16, torch.float32), "q")
    if q.dim() != 4:
        raise SEngineError(f"q: expected (B, L, heads, d), got {tuple(q.shape)}")
    B, L, Hq, d = q.shape
    Hk = 0
    if k is not None:
        _token_input(k, "k", dev)
        if k.dtype != q.dtype or k.dim() != 4 or k.shape[:2] != q.shape[:2] or k.shape[3] != d:
            raise SEngineError(f"k: expected {q.dtype} ({B}, {L}, heads, {d}), got {k.dtype} {tuple(k.shape)}")
        Hk = k.shape[2]
    elif out_k is not None:
        raise SEngineError("out_k: there is no k")
    if not 1 <= len(sections) <= 4 or any(type(n) is not int or n < 0 for n in sections):
        raise SEngineError(f"sections: expected 1 to 4 numbers of pairs, got {sections!r}")
    _token_sizes("rotary: B, L, heads, d and sections", B, L, Hq, Hk, d, *sections)
    pairs, axes = sum(sections), len(sections)
    _token_vector(frequencies, pairs, "frequencies", dev)
    _type_code(frequencies, (torch.float32,), "frequencies")
    _token_input(positions, "positions", dev)
    if positions.dtype not in (torch.int32, torch.float32):
        raise SEngineError(f"positions: expected dtype torch.int32 or torch.float32, got {positions.dtype}")
    if tuple(positions.shape) not in ((B, L, axes), (L, axes)) or (axes > 1 and positions.stride(-1) != 1):
        raise SEngineError(f"positions: expected ({B}, {L}, {axes}) or ({L}, {axes}) with a token's axes side by side, got "
                           f"{tuple(positions.shape)}")
    ps = positions.stride() if positions.dim() == 3 else (0, *positions.stride())
    for t, x, name in ((out_q, q, "out_q"), (out_k, k, "out_k")):
        if t is not None:
            _heads_out(t, x.shape, q.dtype, name, dev)
    dense = lambda n: (ctypes.c_int64 * 3)(L * n * d, n * d, d)
    zero = (ctypes.c_int64 * 3)()
    desc = ctypes.byref(RotaryDesc(
        _head_strides(q, "q"), zero if k is None else _head_strides(k, "k"),
        dense(Hq) if out_q is None else _head_strides(out_q, "out_q"),
        dense(Hk) if out_k is None else _head_strides(out_k, "out_k"), (ctypes.c_int64 * 2)(*ps[:2]), B, L, Hq, Hk, d,
        axes, (ctypes.c_int32 * 4)(*sections), code, positions.dtype is torch.float32, bool(interleaved)))
    return _remember(key, (desc, dev))


def rotary(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, frequencies: torch.Tensor, sections,
           interleaved: bool = False, out_q: Optional[torch.Tensor] = None, out_k: Optional[torch.Tensor] = None):
    """Rotary positions with several axes (time, height, width) on queries q (B, L, Hq, d) and keys k (B, L, Hk, d) or
    None; fp16, bf16 or fp32.  Returns (q', k') in their type, k' None without k.

    The first 2 P values of a head are P = sum(sections) pairs, (x[j], x[P + j]), or (x[2 j], x[2 j + 1]) with
    interleaved; the first sections[0] pairs belong to the first axis, and so on (1 to 4 axes).  Pair j turns by
    positions[b, t, axis] * frequencies[j] radians: (x0, x1) -> (x0 cos - x1 sin, x0 sin + x1 cos).  The values behind
    the pairs are copied.  positions (B, L, axes), or (L, axes) for all sequences, int32 or fp32; frequencies (P,)
    fp32.  The angle is formed and reduced in 64 bits, so that far positions turn as near ones do; sines, cosines and
    products are fp32, with one rounding at the end.  Any strides whose heads' d values lie side by side (d <= 1024, a
    token's heads together up to 65536 values).  out_q may be q and out_k k; otherwise they share no memory with an
    input."""
    if _dispatch_modes() or forward_ad._current_level >= 0:
        _token_modes(q, k, positions, frequencies)
    if type(sections) is not tuple:
        sections = tuple(sections)
    key = None
    # 8.0 and True would find the calls of 8 and 1
    if out_q is None and out_k is None and {*map(type, sections)} == {int}:
        try:
            key = ("rotary", q.dtype, q.shape, q.stride(), q.device, _layout(k), positions.dtype, positions.shape,
                   positions.stride(), positions.device, frequencies.dtype, frequencies.shape, frequencies.stride(),
                   frequencies.device, sections, bool(interleaved))
        except AttributeError:
            pass  # not a tensor: the checks say so
    plan = _TOKEN_PLANS.get(key)
    if plan is None or (torch.is_grad_enabled() and (
            q.requires_grad or positions.requires_grad or frequencies.requires_grad
            or (k is not None and k.requires_grad))):
        plan = _rotary_plan(key, q, k, positions, frequencies, sections, interleaved, out_q, out_k)
    desc, dev = plan
    if out_q is None:
        out_q = torch.empty_like(q, memory_format=torch.contiguous_format)
    if out_k is None and k is not None:
        out_k = torch.empty_like(k, memory_format=torch.contiguous_format)
    _launch(_lib.load().sengine_amd_rotary, dev, "rotary", desc, q.data_ptr(), _ptr(k), positions.data_ptr(),
            frequencies.data_ptr(), out_q.data_ptr(), _ptr(out_k))
    return out_q, out_k


# Types of two e2m1 codes a byte: plain bytes, and torch's own where it has one.
_E2M1_BYTES = tuple(t for t in (torch.uint8, getattr(torch, "float4_e2m1fn_x2", None)) if t is not None)


def _linear_e2m1_plan(key, x, weight, group_scale, row_scale, bias, activation, residual, out_dtype, out):
    """(descriptor, bytes of scratch memory, output's shape and type, device) of a checked call."""
    _token_input(x, "x")
    dev, code = x.device, _type_code(x, (torch.float16, torch.bfloat16), "x")
    _token_input(weight, "weight", dev)
    if x.dim() == 0 or weight.dim() != 2 or weight.dtype not in _E2M1_BYTES or 2 * weight.shape[1] != x.shape[-1]:
        raise SEngineError(f"weight: expected e2m1 codes (N, K / 2), two a byte, for x {tuple(x.shape)}, got {weight.dtype} "
                           f"{tuple(weight.shape)}")
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {sorted(ACTIVATIONS)}, got {activation!r}")
    N, K = weight.shape[0], x.shape[-1]
    _token_sizes("linear_e2m1: N and K", N, K)
    _token_input(group_scale, "group_scale", dev)
    _type_code(group_scale, (torch.float8_e4m3fn,), "group_scale")
    group = next((g for g in (32, 64, 128) if tuple(group_scale.shape) == (N, -(-K // g))), 0)
    if not group:
        raise SEngineError(f"group_scale: expected ({N}, K / group) with groups of 32, 64 or 128 of {K} values, got "
                           f"{tuple(group_scale.shape)}")
    M, xs = _token_rows(x, "x")
    wst, sst = _token_rows(weight, "weight")[1], _token_rows(group_scale, "group_scale")[1]
    if out_dtype is None:
        out_dtype = x.dtype
    ocode = _TOKEN_TYPES.get(out_dtype, ENC_E4M3)
    if ocode == ENC_E4M3:
        raise SEngineError(f"out_dtype: expected float16, bfloat16 or float32, got {out_dtype}")
    if row_scale is not None:
        _token_vector(row_scale, N, "row_scale", dev)
        _type_code(row_scale, (torch.float32,), "row_scale")
    bcode = 0
    if bias is not None:
        _token_vector(bias, N, "bias", dev)
        bcode = _type_code(bias, (torch.float16, torch.bfloat16, torch.float32), "bias")
    shape = (*x.shape[:-1], N)
    rs = 0
    if residual is not None:
        _token_input(residual, "residual", dev)
        if residual.shape != shape or residual.dtype != out_dtype:
            raise SEngineError(f"residual: expected {out_dtype} {shape}, got {residual.dtype} "
                               f"{tuple(residual.shape)}")
        rs = _token_rows(residual, "residual")[1]
    os_ = N if out is None else _token_out(out, shape, out_dtype, "out", dev)
    desc = ctypes.byref(LinearE2m1Desc(M, xs, wst, sst, rs, os_, N, K, group, code, ocode, bcode,
                                       ACTIVATIONS[activation]))
    size = ctypes.c_size_t()
    check(_lib.load().sengine_amd_linear_e2m1_workspace(desc, ctypes.byref(size)), "linear_e2m1")
    return _remember(key, (desc, size.value, shape, out_dtype, dev))


def linear_e2m1(x: torch.Tensor, weight: torch.Tensor, group_scale: torch.Tensor,
                row_scale: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, activation: str = "none",
                residual: Optional[torch.Tensor] = None, out_dtype: Optional[torch.dtype] = None,
                out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """act(x w^T + bias) + residual of token rows x (..., K), fp16 or bf16, with a weight (N, K) in 4 bits:
    w[n, k] = row_scale[n] group_scale[n, k // group] code[n, k].

    weight holds the codes, e2m1 (0, 0.5, 1, 1.5, 2, 3, 4, 6 and, with the highest bit, their negatives), two a byte and
    the lower half first: (N, K / 2) uint8 or float4_e2m1fn_x2, K even.  group_scale is (N, ceil(K / group))
    float8_e4m3fn with groups of 32, 64 or 128 values, row_scale (N,) fp32, 1 where None; token_reader.e2m1_groups makes
    the three of a weight.  Nothing of the weight is rounded: a code times a group's scale is a 16-bit value; sums and
    what follows them are fp32, and the result is rounded once to out_dtype (x's type by default; fp16, bf16 or fp32).
    activation, bias, residual and out as linear's.  Up to 64 token rows, and more of narrow weights, read the codes as
    they are; beyond, they are multiplied with the weight widened to 16 bits in scratch memory of torch's allocator."""
    if _dispatch_modes() or forward_ad._current_level >= 0:
        _token_modes(x, weight, group_scale, row_scale, bias, residual)
    key = None
    if out is None:
        try:
            key = ("linear_e2m1", x.dtype, x.shape, x.stride(), x.device, weight.dtype, weight.shape, weight.stride(),
                   weight.device, _layout(group_scale), _layout(row_scale), activation, out_dtype, _layout(bias),
                   _layout(residual))
        except AttributeError:
            pass  # not a tensor: the checks say so
    plan = _TOKEN_PLANS.get(key)
    if plan is None or (torch.is_grad_enabled() and (
            x.requires_grad or group_scale.requires_grad
            or (row_scale is not None and row_scale.requires_grad) or (bias is not None and bias.requires_grad)
            or (residual is not None and residual.requires_grad))):
        plan = _linear_e2m1_plan(key, x, weight, group_scale, row_scale, bias, activation, residual, out_dtype, out)
    desc, size, shape, out_dtype, dev = plan
    if out is None:
        out = x.new_empty(shape) if out_dtype is x.dtype else torch.empty(shape, dtype=out_dtype, device=dev)
    ws = torch.empty(size, dtype=torch.uint8, device=dev) if size else None
    _launch(_lib.load().sengine_amd_linear_e2m1_ws, dev, "linear_e2m1", desc, x.data_ptr(), weight.data_ptr(),
            group_scale.data_ptr(), _ptr(row_scale), _ptr(bias), _ptr(residual), out.data_ptr(), _ptr(ws), size)
    return out


def _decay_plan(key, q, k, v, decay, state, lengths, scale, out, state_out):
    """(descriptor, bytes of scratch memory, states' shape, device) of a checked call."""
    _token_input(q, "q")
    dev, code = q.device, _type_code(q, (torch.float16, torch.bfloat16), "q")
    for t, name in ((k, "k"), (v, "v")):
        _token_input(t, name, dev)
        if t.dtype != q.dtype:
            raise SEngineError(f"{name}: expected {q.dtype}, got {t.dtype}")
    if q.dim() != 4 or k.shape != q.shape or v.dim() != 4 or v.shape[:3] != q.shape[:3]:
        raise SEngineError(f"decay_attention: expected q, k (B, L, H, dk) and v (B, L, H, dv), got {tuple(q.shape)}, "
                           f"{tuple(k.shape)}, {tuple(v.shape)}")
    (B, L, H, dk), dv = q.shape, v.shape[3]
    _token_sizes("decay_attention: B, L, heads, dk and dv", B, L, H, dk, dv)
    _token_vector(decay, H, "decay", dev)
    _type_code(decay, (torch.float32,), "decay")
    if lengths is not None:
        _token_vector(lengths, B, "lengths", dev)
        if lengths.dtype != torch.int32:
            raise SEngineError(f"lengths: expected dtype torch.int32, got {lengths.dtype}")
    matrices = (B, H, dk, dv)
    strides = []
    for t, x, name in ((q, q, "q"), (k, k, "k"), (v, v, "v"), (out, v, "out")):
        if name == "out":
            if t is None:
                strides.append((ctypes.c_int64 * 3)(L * H * dv, H * dv, dv))
                continue
            _heads_out(t, x.shape, q.dtype, name, dev)
        strides.append(_head_strides(t, name))
        if t.numel() and any(n > 1 and s % 8 for n, s in zip(t.shape, strides[-1])):
            raise SEngineError(f"{name}: rows must begin at multiples of 16 bytes (strides {t.stride()})")
    for t, name in ((state, "state"), (state_out, "state_out")):
        if t is None:
            strides.append((ctypes.c_int64 * 2)(*((H * dk * dv, dk * dv) if name == "state_out" else (0, 0))))
            continue
        if name == "state":
            _token_input(t, name, dev)
        else:
            _heads_out(t, matrices, torch.float32, name, dev)
        if t.dtype != torch.float32 or tuple(t.shape) != matrices:
            raise SEngineError(f"{name}: expected torch.float32 {matrices}, got {t.dtype} {tuple(t.shape)}")
        s = t.stride()
        if t.numel() and ((dv > 1 and s[3] != 1) or (dk > 1 and s[2] != dv) or (B > 1 and s[0] % 4) or (H > 1 and s[1] % 4)):
            raise SEngineError(f"{name}: its matrices must be contiguous and begin at multiples of 16 bytes (strides {s})")
        strides.append((ctypes.c_int64 * 2)(*(x if n > 1 else 0 for n, x in zip(matrices, s[:2]))))
    desc = ctypes.byref(DecayDesc(*strides, B, L, H, dk, dv, code, 1.0 / math.sqrt(dk) if scale is None else scale))
    size = ctypes.c_size_t()
    check(_lib.load().sengine_amd_decay_attention_workspace(desc, ctypes.byref(size)), "decay_attention")
    return _remember(key, (desc, size.value, matrices, dev))


def decay_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, decay: torch.Tensor,
                    state: Optional[torch.Tensor] = None, lengths: Optional[torch.Tensor] = None,
                    scale: Optional[float] = None, out: Optional[torch.Tensor] = None,
                    state_out: Optional[torch.Tensor] = None):
    """Causal linear attention with a decay a head: S_t = decay[h] S_{t-1} + k_t^T v_t, o_t = scale q_t S_t.  Returns
    (o, S), o (B, L, H, dv) in q's type and the state behind each sequence's last token (B, H, dk, dv), fp32.

    q and k are (B, L, H, dk), v is (B, L, H, dv), fp16 or bf16; dk is a multiple of 8 up to 128, dv of 8 up to 256; scale
    1 / sqrt(dk) by default.  decay (H,) fp32 in 0..1: the leak of a head's state a token.  state (B, H, dk, dv) fp32 is
    what the sequences begin with, zeros where None: a prompt is one call, and its state the next call's, of a token or of
    many.  lengths (B,) int32: the tokens of each sequence (clamped to 0..L); what lies behind them is not used, its
    outputs are zeros and leave the state alone.  Any strides whose rows are contiguous and begin at multiples of 16
    bytes.  The state and all sums are fp32; more than 16 tokens are matrix products of 16-bit operands, which hold
    what is not 16-bit by itself as sums of two or three: state and additions to it with all of their bits in bf16 and 22 in
    fp16, the weights within 64 tokens with 16.  A value of v that is not finite reaches the outputs
    from its own token on.  `state_out` may be `state`, updated in place; otherwise outputs share no memory with inputs.
    Few heads of many tokens are computed in segments through scratch memory of torch's allocator, joined in a fixed
    order."""
    if _dispatch_modes() or forward_ad._current_level >= 0:
        _token_modes(q, k, v, decay, state, scale)
    if scale is not None and type(scale) is not float:
        scale = _token_number(scale, "scale")
    key = None
    if out is None and state_out is None:
        try:
            key = ("decay", q.dtype, q.shape, q.stride(), q.device, k.dtype, k.shape, k.stride(), k.device, v.dtype,
                   v.shape, v.stride(), v.device, _layout(decay), _layout(state), _layout(lengths), scale)
        except AttributeError:
            pass  # not a tensor: the checks say so
    plan = _TOKEN_PLANS.get(key)
    if plan is None or (torch.is_grad_enabled() and (
            q.requires_grad or k.requires_grad or v.requires_grad or decay.requires_grad
            or (state is not None and state.requires_grad))):
        plan = _decay_plan(key, q, k, v, decay, state, lengths, scale, out, state_out)
    desc, size, matrices, dev = plan
    if out is None:
        out = torch.empty_like(v, memory_format=torch.contiguous_format)
    if state_out is None:
        state_out = (torch.empty(matrices, dtype=torch.float32, device=dev) if state is None
                     else torch.empty_like(state, memory_format=torch.contiguous_format))
    pointers = qp, kp, vp, op, sp, tp = (q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), _ptr(state) or 0,
                                         state_out.data_ptr())
    if (qp | kp | vp | op | sp | tp) & 15:
        for x, t, name in zip(pointers, (q, k, v, out, state, state_out), ("q", "k", "v", "out", "state", "state_out")):
            if x & 15 and t.numel():
                raise SEngineError(f"{name}: must begin at a multiple of 16 bytes")
    ws = torch.empty(size, dtype=torch.uint8, device=dev) if size else None
    _launch(_lib.load().sengine_amd_decay_attention_ws, dev, "decay_attention", desc, qp, kp, vp, decay.data_ptr(),
            sp or None, _ptr(lengths), op, tp, _ptr(ws), size)
    return out, state_out
