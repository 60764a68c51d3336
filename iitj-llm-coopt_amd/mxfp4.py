"""Microscaled 4-bit rows (the OCP format MXFP4) and weights, on gfx950 kernels.

  quantize_mxfp4(x) / dequantize_mxfp4(codes, scales, dtype)   the codec, beside quantize / dequantize
  pack_mxfp4_weight(codes, scales, activations)                a weight for fused.linear
  quantize_mxfp4_weight(weight, activations)                   the same from a bf16 weight

A row of K elements (K a multiple of 32) is K / 2 code bytes, the even element in the low half, and K / 32
scale bytes.  A code is a sign and one of 0, 0.5, 1, 1.5, 2, 3, 4, 6; an element is code * 2^(s - 127) with its
block's scale byte s, NaN where s is 255.  Quantisation takes s - 127 = floor(log2 amax) - 2 (at least
-127) and the nearest code, ties to the even one, 6 for everything above; a block that is not finite gets 255.
Scales that others made may be 253 or 254, which quantisation never gives: their values from 2^128 on are past bf16
and fp32, and are infinities in dequantize_mxfp4 and in products with bf16 rows (in products of 4-bit rows they
are not).
The reference has no such weights; its codes for swapped caches are kv_cache.quantize's.
"""
import ctypes

import torch

from . import _lib

__all__ = ["quantize_mxfp4", "dequantize_mxfp4", "MXFP4Weight", "pack_mxfp4_weight",
           "quantize_mxfp4_weight"]

BLOCK = 32
MAX_ROWS, MAX_N, MAX_K = 1 << 19, 1 << 24, 1 << 22   # of a product


def _aligned(t, nbytes):
    """Contiguous, at an address that is a multiple of nbytes."""
    t = t.contiguous()
    return t if t.data_ptr() % nbytes == 0 else t.clone()


_KINDS = {torch.bfloat16: _lib.DT_BF16, torch.float16: _lib.DT_F16, torch.float32: _lib.DT_F32}


def quantize_mxfp4(x: torch.Tensor):
    """x [..., K] (bf16, fp16 or fp32) -> (codes uint8 [..., K / 2], scales uint8 [..., K / 32])."""
    index = x.get_device()
    if index < 0:
        _lib.require_cuda(x)
    kind = _KINDS.get(x.dtype)
    if kind is None:
        raise ValueError(f"x must be bf16, fp16 or fp32, got {x.dtype}")
    shape = x.shape
    K = shape[-1] if shape else 1
    if K % BLOCK or K >> 31:
        raise ValueError(f"the last dimension must be a multiple of {BLOCK} below 2^31, got {tuple(shape)}")
    if not x.is_contiguous() or x.data_ptr() % 16:
        x = _aligned(x, 16)
    lead = shape[:-1]
    codes = x.new_empty((*lead, K // 2), dtype=torch.uint8)
    scales = x.new_empty((*lead, K // BLOCK), dtype=torch.uint8)
    rows = x.numel() // K if K else 0
    _lib.check(_lib.call_on(index, _lib.entry("coopt_mxfp4_quantize"), kind, x.data_ptr(), rows, K, codes.data_ptr(),
                            scales.data_ptr(), _lib.raw_stream(index)), "coopt_mxfp4_quantize")
    return codes, scales


def _check_rows(codes, scales):
    """K of codes [..., K / 2] and scales [..., K / 32]."""
    cs, ss = codes.shape, scales.shape
    if codes.dtype is not torch.uint8 or scales.dtype is not torch.uint8:
        raise ValueError("codes and scales must be uint8")
    if not cs or len(ss) != len(cs) or cs[:-1] != ss[:-1] or cs[-1] != ss[-1] * (BLOCK // 2):
        raise ValueError(f"codes [..., K / 2] and scales [..., K / {BLOCK}] disagree: {tuple(cs)}, {tuple(ss)}")
    if cs[-1] >> 30:
        raise ValueError(f"rows of less than 2^31 elements, got {2 * cs[-1]}")
    return 2 * cs[-1]


def dequantize_mxfp4(codes: torch.Tensor, scales: torch.Tensor, dtype=torch.bfloat16):
    """The values [..., K] of 4-bit rows: exact in bf16 and fp32 (infinity from 2^128 on), rounded in fp16."""
    index = codes.get_device()
    if index < 0 or index != scales.get_device():
        _lib.require_one_device(codes, scales)
    K = _check_rows(codes, scales)
    kind = _KINDS.get(dtype)
    if kind is None:
        raise ValueError(f"dtype must be bf16, fp16 or fp32, got {dtype}")
    if not codes.is_contiguous() or codes.data_ptr() % 4:
        codes = _aligned(codes, 4)
    if not scales.is_contiguous():
        scales = scales.contiguous()
    out = codes.new_empty((*codes.shape[:-1], K), dtype=dtype)
    rows = out.numel() // K if K else 0
    _lib.check(_lib.call_on(index, _lib.entry("coopt_mxfp4_dequantize"), codes.data_ptr(), scales.data_ptr(), rows, K,
                            kind, out.data_ptr(), _lib.raw_stream(index)), "coopt_mxfp4_dequantize")
    return out


def _check_weight(codes, scales):
    """(N, K) of a weight's codes [N, K / 2] and scales [N, K / 32]."""
    if codes.dim() != 2:
        raise ValueError(f"codes must be [N, K / 2], got {tuple(codes.shape)}")
    N, K = codes.shape[0], _check_rows(codes, scales)
    if N > MAX_N or K > MAX_K:
        raise ValueError(f"a weight of at most {MAX_N} x {MAX_K}, got {N} x {K}")
    return N, K


def _check_activations(activations):
    if activations not in ("bf16", "mxfp4"):
        raise ValueError(f"activations must be 'bf16' or 'mxfp4', got {activations!r}")


class MXFP4Weight:
    """A projection weight [N, K] in microscaled 4 bits: `codes` and `scales` as they were given, and
    `packed`, the copy that fused.linear streams (coopt_mxfp4_pack_weight's layout; it does not see
    later changes of the codes).

    activations "bf16": products with the rows as they are.  "mxfp4": rows are quantised to 4 bits in the call and
    both operands go to the scaled matrix instructions (4 bits by 4 bits)."""

    def __init__(self, codes, scales, packed, activations="bf16"):
        _check_activations(activations)
        N, K = _check_weight(codes, scales)
        if not codes.device == scales.device == packed.device:
            raise ValueError(f"codes, scales and packed on {codes.device}, {scales.device}, {packed.device}: one device "
                             "is needed")
        size = int(_lib.entry("coopt_mxfp4_packed_bytes")(N, K))   # the kernels read all of it
        if packed.dtype is not torch.uint8 or packed.numel() != size or not packed.is_contiguous() or \
                packed.data_ptr() % 16:
            raise ValueError(f"packed must be {size} contiguous bytes (uint8), 16-byte aligned")
        self.codes, self.scales, self.packed, self.activations = codes, scales, packed, activations
        self.shape = torch.Size((N, K))
        self.act4 = 1 if activations == "mxfp4" else 0
        self._plans = {}   # rows: what plan() returns, a pure function of the sizes

    def plan(self, rows):
        """(workspace bytes, K slices a consumer would add, padded rows and workspace bytes of those) of a
        product of `rows` rows."""
        p = self._plans.get(rows)
        if p is None:
            if rows > MAX_ROWS:
                raise ValueError(f"at most {MAX_ROWS} rows, got {rows}")
            lib, (N, K) = _lib.load(), self.shape
            ks, padded = ctypes.c_int(0), ctypes.c_int(0)
            _lib.check(lib.coopt_mxfp4_linear_split(rows, N, K, self.act4, ctypes.byref(ks), ctypes.byref(padded)),
                       "coopt_mxfp4_linear_split")
            size = lib.coopt_mxfp4_linear_workspace
            p = (int(size(rows, N, K, self.act4, 0)), ks.value if N % 32 == 0 else 1, padded.value,
                 int(size(rows, N, K, self.act4, 1)))
            if len(self._plans) >= 4096:
                self._plans.clear()
            self._plans[rows] = p
        return p

    @property
    def dtype(self):
        return torch.bfloat16   # of the values it stands for

    @property
    def device(self):
        return self.codes.device

    def dequantize(self, dtype=torch.bfloat16):
        """The values [N, K], row-major."""
        return dequantize_mxfp4(self.codes, self.scales, dtype)


def pack_mxfp4_weight(codes, scales, activations="bf16"):
    """MXFP4Weight of codes [N, K / 2] and scales [N, K / 32] on the GPU: one launch at model load."""
    _check_activations(activations)
    index = codes.get_device()
    if index < 0 or index != scales.get_device():
        _lib.require_one_device(codes, scales)
    N, K = _check_weight(codes, scales)
    cc, sc = _aligned(codes, 16), scales.contiguous()
    nbytes = int(_lib.entry("coopt_mxfp4_packed_bytes")(N, K))
    packed = cc.new_empty(nbytes)
    _lib.check(_lib.call_on(index, _lib.entry("coopt_mxfp4_pack_weight"), cc.data_ptr(), sc.data_ptr(), N, K,
                            packed.data_ptr(), _lib.raw_stream(index)), "coopt_mxfp4_pack_weight")
    return MXFP4Weight(cc, sc, packed, activations)


def quantize_mxfp4_weight(weight, activations="bf16"):
    """MXFP4Weight of a weight [N, K] on the GPU, quantised by quantize_mxfp4."""
    if weight.dim() != 2:
        raise ValueError(f"weight must be [N, K], got {tuple(weight.shape)}")
    return pack_mxfp4_weight(*quantize_mxfp4(weight), activations=activations)
