"""Paged KV cache writes and the symmetric absmax INT8/INT4 codec, on gfx950 kernels.

Drop-in surfaces (reference paths under mohsinmubarak/iitj-llm-coopt):
  quantize(x, bits) / dequantize(q, scale, bits, dtype)   engine/kv_tier_manager.py:21-41
  reshape_and_cache_flash(k, v, k_cache, v_cache, slot_mapping, kv_cache_dtype, k_scale,
                          v_scale)                         engine/model.py:242-243 (vLLM op)
  qkv_rope_and_cache(qkv, positions, cos, sin, ...)        engine/model.py:238-243 in one launch
  qkv_norm_rope_and_cache(qkv, q_weight, k_weight, ...)    the same with normed q and k heads

Cache layouts.  bf16 ("auto"): k_cache/v_cache [num_blocks, block_size, Hkv, D] bf16, possibly
a strided per-layer view of a block-major buffer (engine/elastic.py:74-77).  INT8 ("int8"):
int8 codes of the same shape plus fp16 scales [num_blocks, block_size, Hkv] passed as
k_scale/v_scale -- per (token, head) vector, exactly what quantize(cache[blocks], 8) produces
(engine/kv_tier_manager.py:99; SwappedKV shapes :46-49).  INT4 ("int4"): uint8 [num_blocks,
block_size, Hkv, D/2], two codes a byte, with the same scales: what quantize(cache[blocks], 4)
produces.
"""
import torch

from . import _lib
from .fused import LinearPartials

__all__ = ["quantize", "dequantize", "reshape_and_cache_flash", "allocate_kv_cache",
           "qkv_rope_and_cache", "qkv_norm_rope_and_cache"]


def quantize(x: torch.Tensor, bits: int):
    """x [..., D] -> (q, scale [...]) with symmetric absmax per last-dim vector.

    bits 16 returns (x.clone(), None) like the reference; bits 8 gives int8 codes; bits 4 packs
    two signed nibbles (+8 offset) per uint8, even element in the low nibble.
    """
    if bits == 16:
        return x.clone(), None
    if bits not in (8, 4):
        raise ValueError(f"bits must be 16, 8 or 4, got {bits}")
    _lib.require_cuda(x)
    D = x.shape[-1]
    xc = x.contiguous()
    rows = xc.numel() // D if D else 0
    if bits == 8:
        q = torch.empty(x.shape, dtype=torch.int8, device=x.device)
    else:
        if D % 2:
            raise ValueError("INT4 packing needs an even last dimension")
        q = torch.empty((*x.shape[:-1], D // 2), dtype=torch.uint8, device=x.device)
    scale = torch.empty(x.shape[:-1], dtype=torch.float16, device=x.device)
    lib = _lib.load()
    _lib.check(lib.coopt_quantize(bits, _lib.dt_code(x.dtype), _lib.ptr(xc), rows, D,
                                  _lib.ptr(q), _lib.ptr(scale), _lib.stream_handle(x.device)),
               "coopt_quantize")
    return q, scale


def dequantize(q: torch.Tensor, scale, bits: int, dtype=torch.bfloat16):
    """Inverse of quantize: dtype(float(code) * float(scale)) per element."""
    if bits == 16:
        return q
    if bits not in (8, 4):
        raise ValueError(f"bits must be 16, 8 or 4, got {bits}")
    index = q.get_device()
    if index < 0 or index != scale.get_device():
        _lib.require_one_device(q, scale)
    qc, sc = q.contiguous(), scale.contiguous()
    *lead, width = qc.shape
    D = width * (2 if bits == 4 else 1)
    if sc.numel() * width != qc.numel():
        raise ValueError(f"scale must have one entry a vector, shape {tuple(lead)}, got {tuple(scale.shape)}")
    out = qc.new_empty((*lead, D), dtype=dtype)
    _lib.check(_lib.call_on(index, _lib.entry("coopt_dequantize"), bits, qc.data_ptr(), sc.data_ptr(),
                            sc.numel(), D, _lib.dt_code(dtype), out.data_ptr(), _lib.raw_stream(index)),
               "coopt_dequantize")
    return out


def allocate_kv_cache(num_blocks: int, block_size: int, num_kv_heads: int, head_dim: int,
                      kv_cache_dtype: str = "auto", device="cuda", dtype=torch.bfloat16):
    """One layer's (k_cache, v_cache, k_scale, v_scale); the scales are None for "auto".

    Every tensor has the reference's logical shape -- caches [num_blocks, block_size, Hkv, D]
    (engine/model.py:148-155), INT8 scales [num_blocks, block_size, Hkv] -- as a view of
    head-major storage [num_blocks, Hkv, block_size, ...]: one head's tokens of a block are
    adjacent in HBM, so the verify-attention kernel reads each (block, head) as one contiguous
    run (16 tokens x D codes) instead of D-sized pieces strided by Hkv * D.  The kernels take
    any strides, so caches in the reference's token-major layout work too.
    """
    store = (num_blocks, num_kv_heads, block_size, head_dim)
    if kv_cache_dtype == "auto":
        return (torch.zeros(store, dtype=dtype, device=device).transpose(1, 2),
                torch.zeros(store, dtype=dtype, device=device).transpose(1, 2), None, None)
    if kv_cache_dtype == "int8":
        sstore = (num_blocks, num_kv_heads, block_size)
        return (torch.zeros(store, dtype=torch.int8, device=device).transpose(1, 2),
                torch.zeros(store, dtype=torch.int8, device=device).transpose(1, 2),
                torch.zeros(sstore, dtype=torch.float16, device=device).transpose(1, 2),
                torch.zeros(sstore, dtype=torch.float16, device=device).transpose(1, 2))
    if kv_cache_dtype == "int4":
        if head_dim % 2:
            raise ValueError("'int4' caches need an even head_dim")
        store = (num_blocks, num_kv_heads, block_size, head_dim // 2)
        # zeros, as in the other caches: two codes of 0, offset by +8
        return (torch.full(store, 0x88, dtype=torch.uint8, device=device).transpose(1, 2),
                torch.full(store, 0x88, dtype=torch.uint8, device=device).transpose(1, 2),
                torch.zeros(store[:3], dtype=torch.float16, device=device).transpose(1, 2),
                torch.zeros(store[:3], dtype=torch.float16, device=device).transpose(1, 2))
    raise ValueError(f"kv_cache_dtype must be 'auto', 'int8' or 'int4', got {kv_cache_dtype!r}")


def _scale_args(k_cache, k_scale, v_scale, kv_cache_dtype):
    """The strides of the scale caches of an "int8" or "int4" cache, checked."""
    if k_scale is None or v_scale is None:
        raise ValueError(f"{kv_cache_dtype!r} caches need k_scale and v_scale scale caches")
    if k_scale.shape != k_cache.shape[:3] or k_scale.dtype != torch.float16 or \
            v_scale.dtype != torch.float16 or k_scale.stride() != v_scale.stride() or \
            v_scale.shape != k_scale.shape:
        raise ValueError("scale caches must be fp16 [num_blocks, block_size, Hkv] alike")
    return k_scale.stride()


def _check_int4(k_cache, v_cache):
    if k_cache.dtype != torch.uint8 or v_cache.dtype != torch.uint8:
        raise ValueError("'int4' caches hold two codes a byte in uint8")


def _check_cache_pair(k_cache, v_cache):
    if k_cache.shape != v_cache.shape or k_cache.stride() != v_cache.stride():
        raise ValueError("k_cache and v_cache must have the same shape and strides")
    if k_cache.dim() != 4 or k_cache.stride(-1) != 1:
        raise ValueError("caches must be [num_blocks, block_size, Hkv, D] with contiguous D")


def reshape_and_cache_flash(k, v, k_cache, v_cache, slot_mapping, kv_cache_dtype="auto",
                            k_scale=None, v_scale=None):
    """k_cache[slot // bs, slot % bs] = k (and v), in place; slots < 0 are skipped.

    kv_cache_dtype "auto": bf16 caches, k_scale/v_scale ignored (the reference passes fp32
    ones, engine/model.py:129).  "int8": int8 code caches; k_scale/v_scale are the fp16
    [num_blocks, block_size, Hkv] scale caches and each written vector is quantised in the
    same kernel.  "int4": the same with uint8 caches of two codes a byte.
    Tokens of one call have slots of their own: of two with the same, either's codes and either's
    scale may stay.
    """
    # get_device() is -1 on the CPU; 0.04 us, a device object twice that
    index = k.get_device()
    alike = index >= 0 and index == v.get_device() == k_cache.get_device() == \
        v_cache.get_device() == slot_mapping.get_device()
    if not alike:
        _lib.require_cuda(k, v, k_cache, v_cache, slot_mapping)
    _check_cache_pair(k_cache, v_cache)
    if k.shape != v.shape or k.dim() != 3 or k.stride(-1) != 1 or v.stride(-1) != 1:
        raise ValueError("k and v must be [T, Hkv, D] with contiguous D")
    if k.dtype is not _BF16 or v.dtype is not _BF16:
        raise ValueError("k and v must be bf16")
    T, Hkv, D = k.shape
    NB, bs, cH, cD = k_cache.shape
    if cH != Hkv or cD != (D // 2 if kv_cache_dtype == "int4" else D):
        raise ValueError(f"cache heads/dim {(cH, cD)} != k's {(Hkv, D)}")
    if slot_mapping.dtype is not torch.int64 or slot_mapping.numel() != T:
        raise ValueError("slot_mapping must be int64 with one entry per token")
    if not slot_mapping.is_contiguous():
        slot_mapping = slot_mapping.contiguous()
    if kv_cache_dtype == "auto":
        if k_cache.dtype is not _BF16:
            raise ValueError("'auto' caches are bf16")
        code, ks, vs, sstr = _lib.DT_BF16, 0, 0, (0, 0, 0)
    elif kv_cache_dtype == "int8":
        if k_cache.dtype is not torch.int8:
            raise ValueError("'int8' caches hold int8 codes")
        if k_scale is None or v_scale is None:
            raise ValueError("'int8' caches need k_scale and v_scale scale caches")
        if k_scale.shape != (NB, bs, Hkv) or k_scale.dtype is not torch.float16 or \
                k_scale.stride() != v_scale.stride() or v_scale.shape != k_scale.shape:
            raise ValueError("scale caches must be fp16 [num_blocks, block_size, Hkv] alike")
        _lib.require_cuda(k_scale, v_scale)
        code, ks, vs, sstr = _lib.DT_I8, k_scale.data_ptr(), v_scale.data_ptr(), k_scale.stride()
    elif kv_cache_dtype == "int4":
        _check_int4(k_cache, v_cache)
        sstr = _scale_args(k_cache, k_scale, v_scale, "int4")
        if not (alike and index == k_scale.get_device() == v_scale.get_device()):
            _lib.require_one_device(k, v, k_cache, v_cache, slot_mapping, k_scale, v_scale)
        code, ks, vs = _lib.DT_I4, k_scale.data_ptr(), v_scale.data_ptr()
    else:
        raise ValueError(f"kv_cache_dtype must be 'auto', 'int8' or 'int4', got {kv_cache_dtype!r}")
    c0, c1, c2, _ = k_cache.stride()
    k0, k1, _ = k.stride()
    v0, v1, _ = v.stride()
    _lib.check(_lib.call_on(
        index, _lib.entry("coopt_kv_write"), code, k.data_ptr(), v.data_ptr(), k0, k1, v0, v1,
        k_cache.data_ptr(), v_cache.data_ptr(), c0, c1, c2, ks, vs, sstr[0], sstr[1], sstr[2],
        slot_mapping.data_ptr(), T, Hkv, D, bs, NB, _lib.raw_stream(index)), "coopt_kv_write")


def qkv_rope_and_cache(qkv, positions, cos, sin, k_cache, v_cache, slot_mapping, num_heads,
                       num_kv_heads, head_dim, kv_cache_dtype="auto", k_scale=None,
                       v_scale=None, q_out=None):
    """The chain after the qkv projection (engine/model.py:238-243) in one launch: split q/k/v,
    neox RoPE on q and k, k and v into the paged cache (as reshape_and_cache_flash), and
    return q [T, num_heads, head_dim].  `qkv` is the projection's bf16 output [T, (Hq + 2 Hkv)
    D] or its fused.LinearPartials (split-K partials, reduced here).  Bit for bit the same as
    rope_ + reshape_and_cache_flash on the reduced output."""
    Hq, Hkv, D = int(num_heads), int(num_kv_heads), int(head_dim)
    width = (Hq + 2 * Hkv) * D
    part = qkv if isinstance(qkv, LinearPartials) else None
    if part is not None:
        if part.n != width:
            raise ValueError(f"partials are {part.n} wide, expected {width}")
        T, src, qkv_t = part.rows, part.buf, None
    else:
        _lib.require_cuda(qkv)
        if qkv.dtype != torch.bfloat16 or qkv.dim() != 2 or qkv.shape[1] != width or qkv.stride(1) != 1:
            raise ValueError(f"qkv must be bf16 [T, {width}] with contiguous rows")
        T, src, qkv_t = qkv.shape[0], qkv, qkv
    index = src.get_device()
    if not (index >= 0 and index == positions.get_device() == cos.get_device() == sin.get_device() ==
            k_cache.get_device() == v_cache.get_device() == slot_mapping.get_device() ==
            (index if q_out is None else q_out.get_device())):
        _lib.require_one_device(src, positions, cos, sin, k_cache, v_cache, slot_mapping, q_out)
    _check_cache_pair(k_cache, v_cache)
    NB, bs, cH, cD = k_cache.shape
    if (cH, cD) != (Hkv, D // 2 if kv_cache_dtype == "int4" else D):
        raise ValueError(f"cache heads/dim {(cH, cD)} != ({Hkv}, {D})")
    if slot_mapping.dtype != torch.int64 or slot_mapping.numel() != T:
        raise ValueError("slot_mapping must be int64 with one entry per token")
    if positions.dtype != torch.int64 or positions.numel() != T:
        raise ValueError("positions must be int64 with one entry per token")
    if cos.shape != sin.shape or cos.stride() != sin.stride() or cos.shape[1] < D // 2 or \
            cos.dtype != torch.bfloat16 or cos.stride(1) != 1:
        raise ValueError("cos/sin tables must be bf16 [max_pos, >= D/2] alike")
    if kv_cache_dtype == "auto":
        code, ks, vs, sstr = _lib.DT_BF16, None, None, (0, 0, 0)
    elif kv_cache_dtype == "int8":
        if k_scale is None or v_scale is None or k_scale.stride() != v_scale.stride():
            raise ValueError("'int8' caches need alike k_scale and v_scale scale caches")
        if not index == k_scale.get_device() == v_scale.get_device():
            _lib.require_one_device(k_cache, k_scale, v_scale)
        code, ks, vs, sstr = _lib.DT_I8, k_scale, v_scale, k_scale.stride()
    elif kv_cache_dtype == "int4":
        _check_int4(k_cache, v_cache)
        sstr = _scale_args(k_cache, k_scale, v_scale, "int4")
        if not index == k_scale.get_device() == v_scale.get_device():
            _lib.require_one_device(k_cache, k_scale, v_scale)
        code, ks, vs = _lib.DT_I4, k_scale, v_scale
    else:
        raise ValueError(f"kv_cache_dtype must be 'auto', 'int8' or 'int4', got {kv_cache_dtype!r}")
    if q_out is None:
        q_out = torch.empty((T, Hq, D), dtype=torch.bfloat16, device=src.device)
    positions, slot_mapping = positions.contiguous(), slot_mapping.contiguous()
    cs = k_cache.stride()
    _lib.check(_lib.call_on(
        index, _lib.entry("coopt_qkv_epilogue"), code, _lib.ptr(qkv_t), 0 if qkv_t is None else qkv_t.stride(0),
        None if part is None else _lib.ptr(part.buf), 0 if part is None else part.ks,
        0 if part is None else part.rows_padded * part.n,
        _lib.ptr(positions), _lib.ptr(cos), _lib.ptr(sin), cos.stride(0),
        cos.shape[0], _lib.ptr(q_out), q_out.stride(0), q_out.stride(1), _lib.ptr(k_cache),
        _lib.ptr(v_cache), cs[0], cs[1], cs[2], _lib.ptr(ks), _lib.ptr(vs), sstr[0], sstr[1],
        sstr[2], _lib.ptr(slot_mapping), T, Hq, Hkv, D, bs, NB,
        _lib.raw_stream(index)), "coopt_qkv_epilogue")
    return q_out


_BF16 = torch.bfloat16
_CACHE_KINDS = {"auto": (_lib.DT_BF16, torch.bfloat16, 1), "int8": (_lib.DT_I8, torch.int8, 1),
                "int4": (_lib.DT_I4, torch.uint8, 2)}   # code, type, elements a unit of it holds


def qkv_norm_rope_and_cache(qkv, q_weight, k_weight, eps, positions, cos, sin, k_cache, v_cache,
                            slot_mapping, num_heads, num_kv_heads, head_dim, kv_cache_dtype="auto",
                            k_scale=None, v_scale=None, q_out=None):
    """qkv_rope_and_cache for models that norm their query and key heads: in one launch, every q
    and k head vector x becomes RoPE(x * rsqrt(mean(x^2) + eps) * weight), computed in fp32 and
    rounded to bf16 once; k and v go to the paged cache and q [T, num_heads, head_dim] is returned.

    q_weight, k_weight: bf16 [head_dim].  `qkv` is the projection's bf16 output [T, (Hq + 2 Hkv) D]
    or its fused.LinearPartials.  kv_cache_dtype "auto", "int8" or "int4", as in
    reshape_and_cache_flash; rows with slot < 0 write no cache entry.  head_dim 64, 128 or 256."""
    Hq, Hkv, D = int(num_heads), int(num_kv_heads), int(head_dim)
    part = None
    if isinstance(qkv, LinearPartials):
        part, x, T, width, stride = qkv, qkv.buf, qkv.rows, qkv.n, 0
    else:
        x = qkv
        if x.dim() != 2 or x.dtype is not _BF16:
            raise ValueError("qkv must be bf16 [T, (Hq + 2 Hkv) * D] with contiguous rows")
        T, width = x.shape
        stride, inner = x.stride()
        if inner != 1 and width > 1:
            raise ValueError("qkv must be bf16 [T, (Hq + 2 Hkv) * D] with contiguous rows")
    if width != (Hq + 2 * Hkv) * D:
        raise ValueError(f"qkv must be {(Hq + 2 * Hkv) * D} wide, got {width}")
    kind = _CACHE_KINDS.get(kv_cache_dtype)
    if kind is None:
        raise ValueError(f"kv_cache_dtype must be 'auto', 'int8' or 'int4', got {kv_cache_dtype!r}")
    code, dtype, per_unit = kind
    _check_cache_pair(k_cache, v_cache)
    NB, bs, cH, cD = k_cache.shape
    if cH != Hkv or cD * per_unit != D:
        raise ValueError(f"cache heads/dim {(cH, cD)} != ({Hkv}, {D // per_unit})")
    if k_cache.dtype is not dtype or v_cache.dtype is not dtype:
        raise ValueError(f"{kv_cache_dtype!r} caches hold {dtype}")
    # one GPU for all of them (get_device() is -1 on the CPU; 0.04 us, a device object twice that)
    index = x.get_device()
    alike = index >= 0 and index == k_cache.get_device() == v_cache.get_device() == \
        slot_mapping.get_device() == positions.get_device() == cos.get_device() == \
        sin.get_device() == q_weight.get_device() == k_weight.get_device()
    if code == _lib.DT_BF16:
        ks = vs = s0 = s1 = s2 = 0
    else:
        s0, s1, s2 = _scale_args(k_cache, k_scale, v_scale, kv_cache_dtype)
        alike = alike and index == k_scale.get_device() == v_scale.get_device()
        ks, vs = k_scale.data_ptr(), v_scale.data_ptr()
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w.dtype is not _BF16 or w.dim() != 1 or w.numel() != D or not w.is_contiguous():
            raise ValueError(f"{name} must be bf16 [{D}], contiguous")
    if slot_mapping.dtype is not torch.int64 or slot_mapping.numel() != T:
        raise ValueError("slot_mapping must be int64 with one entry per token")
    if positions.dtype is not torch.int64 or positions.numel() != T:
        raise ValueError("positions must be int64 with one entry per token")
    if cos.dtype is not _BF16 or sin.dtype is not _BF16 or cos.dim() != 2 or cos.shape != sin.shape:
        raise ValueError("cos/sin tables must be bf16 [max_pos, >= D/2] alike")
    rows, half = cos.shape
    tab = cos.stride()
    if tab != sin.stride() or tab[1] != 1 or half < D // 2 or rows < 1:
        raise ValueError("cos/sin tables must be bf16 [max_pos, >= D/2] alike")
    if q_out is not None:
        if q_out.shape != (T, Hq, D) or q_out.dtype is not _BF16 or q_out.stride(-1) != 1:
            raise ValueError("q_out must be bf16 [T, Hq, D] with contiguous D")
        alike = alike and index == q_out.get_device()
    if not alike:
        _lib.require_one_device(x, q_weight, k_weight, positions, cos, sin, k_cache, v_cache, slot_mapping,
                                k_scale if ks else None, v_scale if vs else None, q_out)
    if q_out is None:
        q_out = cos.new_empty((T, Hq, D))
    if T == 0:
        return q_out
    if not positions.is_contiguous():
        positions = positions.contiguous()
    if not slot_mapping.is_contiguous():
        slot_mapping = slot_mapping.contiguous()
    c0, c1, c2, _ = k_cache.stride()
    q0, q1, _ = q_out.stride()
    _lib.check(_lib.call_on(
        index, _lib.entry("coopt_qkv_norm_epilogue"), code, 0 if part is not None else x.data_ptr(), stride,
        0 if part is None else x.data_ptr(), 0 if part is None else part.ks,
        0 if part is None else part.rows_padded * part.n, q_weight.data_ptr(), k_weight.data_ptr(),
        float(eps), positions.data_ptr(), cos.data_ptr(), sin.data_ptr(), tab[0], rows, q_out.data_ptr(), q0,
        q1, k_cache.data_ptr(), v_cache.data_ptr(), c0, c1, c2, ks, vs, s0, s1, s2,
        slot_mapping.data_ptr(), T, Hq, Hkv, D, bs, NB, _lib.raw_stream(index)),
        "coopt_qkv_norm_epilogue")
    return q_out
