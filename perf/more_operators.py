"""Operators of a forward pass with 4-bit weights, as measurable cases.

quant   microscaled 4-bit quantisation of rows, and the values back (quantize_mxfp4, dequantize_mxfp4)
weight  a projection of bf16 rows by a microscaled 4-bit weight (fused.linear)
both    the same with the rows quantised to 4 bits in the call
norm    the norm behind a block, its gate and scale, the residual sum and the next block's norm
        (fused.residual_norm)

`own` false: the plain form, elementary torch operations in 32 bits, rounded once at the end.
`own` true: the calls a serving program makes of this package.  Widths of the listed cases are those of the
package's own 8B and 1B shapes, row counts those of decoding, verification and prompts; `draw` takes the
ranges around them.

A microscaled row holds, for every 32 elements along its length, 32 codes of 4 bits (sign, then
0, 0.5, 1, 1.5, 2, 3, 4, 6; the even element in the low half of its byte) and one byte s: the elements are
code * 2^(s - 127).  For the largest magnitude a of 32 elements, s - 127 = floor(log2 a) - 2, at least -127, and a
code is the nearest one to x / 2^(s - 127), ties to the even code, 6 for all above.

listed() / draw(rng)      cases: dicts of plain values
prepare(case, seed)       inputs and weights a program holds before the call
run(state)                one pass; returns every output
work(case)                bytes and flops the pass cannot do without
exact(case, seed)         the outputs in 64 bits, from the definition
"""
import math

import torch

own = False

DEV = "cuda"
EPS = 1e-5
BLOCK = 32


def listed():
    return [
        # The rows of a verify step on their way into a product of two 4-bit operands.
        dict(name="quant_verify", kind="quant", M=160, K=4096, dtype="bf16"),
        # A whole projection's weight, quantised when a model is loaded.
        dict(name="quant_weight", kind="quant", M=28672, K=4096, dtype="bf16"),
        # One user, one token, the attention's output projection: latency.
        dict(name="weight_decode_b1", kind="weight", M=1, N=4096, K=4096),
        # The draft proposes a token for 32 sequences: its widest layer.
        dict(name="weight_draft", kind="weight", M=32, N=16384, K=2048),
        # A batch that shrank to 77 rows, through the projection with the longest sums.
        dict(name="weight_down_ragged", kind="weight", M=77, N=4096, K=14336),
        # The target verifies 5 rows of 32 sequences: its widest layer.
        dict(name="weight_verify", kind="weight", M=160, N=28672, K=4096),
        # A prompt of 2000 tokens.
        dict(name="weight_prompt", kind="weight", M=2000, N=4096, K=14336),
        # A few sequences decode with both operands in 4 bits.
        dict(name="both_decode", kind="both", M=9, N=2048, K=8192),
        # The verify step's widest layer with both operands in 4 bits.
        dict(name="both_verify", kind="both", M=160, N=28672, K=4096),
        # Prompts admitted together, 4093 tokens in all: the largest product.
        dict(name="both_prompt", kind="both", M=4093, N=28672, K=4096),
        # The norms between two blocks of one token's forward.
        dict(name="norm_decode_b1", kind="norm", T=1, H=4096, gate="channel", post=True),
        # The same for prompts, gated token by token: bandwidth.
        dict(name="norm_prompts", kind="norm", T=8191, H=4096, gate="token", post=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["quant", "weight", "weight", "both", "both", "norm"])
    if kind == "quant":
        return dict(kind=kind, M=_log(rng, 1, 16384), K=BLOCK * _log(rng, 1, 200),
                    dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]))
    if kind == "norm":
        return dict(kind=kind, T=_log(rng, 1, 8191), H=8 * _log(rng, 16, 1000),
                    gate=rng.choice(["none", "channel", "token"]), post=rng.random() < 0.7)
    N, K = _log(rng, 60, 28672), BLOCK * _log(rng, 4, 448)
    top = min(4093, 4 * 10 ** 11 // (N * K))
    M = rng.choice([_log(rng, 1, 256), _log(rng, 1, 4093)])
    return dict(kind=kind, M=max(1, min(M, top)), N=N, K=K)


# ---- inputs ----------------------------------------------------------------------------------

def _randn(g, *size):
    return torch.randn(*size, generator=g, device=DEV)


def _rows(g, M, K):
    """Rows as a norm gives them: 0.5 % of the channels 20 times as large."""
    big = torch.rand(K, generator=g, device=DEV) < 0.005
    return _randn(g, M, K) * torch.where(big, 20.0, 1.0)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    st = dict(case=case)
    kind = case["kind"]
    if kind == "quant":
        dtype = dict(bf16=torch.bfloat16, fp16=torch.float16, fp32=torch.float32)[case["dtype"]]
        st["x"] = _rows(g, case["M"], case["K"]).to(dtype)
    elif kind == "norm":
        T, H = case["T"], case["H"]
        st["x"], st["residual"] = (3 * _randn(g, T, H)).to(torch.bfloat16), (10 * _randn(g, T, H)).to(torch.bfloat16)
        st["weight"], st["post"] = ((1 + 0.3 * _randn(g, H)).to(torch.bfloat16) for _ in range(2))
        st["gate"] = dict(none=None, channel=torch.sigmoid(_randn(g, H)).to(torch.bfloat16),
                          token=torch.sigmoid(_randn(g, T, H)).to(torch.bfloat16)
                          if case["gate"] == "token" else None)[case["gate"]]
        st["post"] = st["post"] if case["post"] else None
        st["scale"], st["new"] = 0.22, torch.empty_like(st["residual"])
    else:
        st["x"] = _rows(g, case["M"], case["K"]).to(torch.bfloat16)
        # weights as they lie in a checkpoint: codes [N, K / 2] and scales [N, K / 32]
        st["codes"], st["scales"] = _quantize(0.02 * _randn(g, case["N"], case["K"]))
        if own:
            import iitj_llm_coopt_amd as M
            st["weight"] = M.pack_mxfp4_weight(st["codes"], st["scales"],
                                               activations="mxfp4" if kind == "both" else "bf16")
    return st


# ---- the plain forms -------------------------------------------------------------------------

_BETWEEN = (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)   # halfway from one code to the next


def _quantize(x):
    """codes [M, K / 2] and scale bytes [M, K / 32] of fp32 x."""
    M, K = x.shape
    y = x.reshape(M, K // BLOCK, BLOCK)
    amax = y.abs().amax(-1)
    e = (torch.frexp(amax).exponent - 3).clamp_min(-127)      # amax = f * 2^exponent, f in [0.5, 1)
    e = torch.where(amax > 0, e, -127)
    y = torch.ldexp(torch.ldexp(y, -(e // 2).unsqueeze(-1)), -(e - e // 2).unsqueeze(-1))
    a = y.abs()
    code = torch.zeros_like(a, dtype=torch.uint8)
    for i, b in enumerate(_BETWEEN):                           # a tie goes to the even code
        code += (a > b) if i % 2 == 0 else (a >= b)
    code |= torch.signbit(y).to(torch.uint8) << 3
    code = code.reshape(M, K // 2, 2)
    return code[..., 0] | (code[..., 1] << 4), (e + 127).to(torch.uint8)


def _values(codes, scales):
    """fp32 [M, K] of codes and scale bytes."""
    table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], device=codes.device)
    table = torch.cat([table, -table])
    x = table[torch.stack([codes & 15, codes >> 4], -1).flatten(-2).int()]
    x = x.reshape(*scales.shape, BLOCK) * torch.exp2(scales.float() - 127).unsqueeze(-1)
    return x.flatten(-2)


def _plain_norm(st):
    case, x = st["case"], st["x"].float()
    if case["post"]:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * st["post"].float()
    if st["gate"] is not None:
        x = x * st["gate"].float()
    r = st["residual"].float() + st["scale"] * x
    out = r * torch.rsqrt((r * r).mean(-1, keepdim=True) + EPS) * st["weight"].float()
    return out.to(torch.bfloat16), r.to(torch.bfloat16)


# ---- one pass --------------------------------------------------------------------------------

def run(st):
    kind = st["case"]["kind"]
    if own:
        import iitj_llm_coopt_amd as M
        if kind == "quant":
            return M.dequantize_mxfp4(*M.quantize_mxfp4(st["x"]))
        if kind == "norm":
            out = M.fused.residual_norm(st["x"], st["residual"], st["weight"], EPS, post_weight=st["post"],
                                        gate=st["gate"], branch_scale=st["scale"], residual_out=st["new"])
            return out, st["new"]
        return M.fused.linear(st["x"], st["weight"])
    if kind == "quant":
        return _values(*_quantize(st["x"].float())).to(torch.bfloat16)
    if kind == "norm":
        return _plain_norm(st)
    x = st["x"].float()
    if kind == "both":
        x = _values(*_quantize(x))
    return torch.matmul(x, _values(st["codes"], st["scales"]).t()).to(torch.bfloat16)


# ---- what a pass cannot do without -----------------------------------------------------------

def work(case):
    kind = case["kind"]
    if kind == "quant":
        # the rows in, codes and scales out and in again, the values out
        n = case["M"] * case["K"]
        return dict(bytes=n * (4 if case["dtype"] == "fp32" else 2) + 2 * n * 17 // 32 + 2 * n, flops=4 * n)
    if kind == "norm":
        T, H, gate = case["T"], case["H"], case["gate"]
        per_channel = 2 + (2 if case["post"] else 0) + (2 if gate == "channel" else 0)
        return dict(bytes=T * H * (8 + (2 if gate == "token" else 0)) + H * per_channel,
                    flops=T * H * (10 if case["post"] else 7))
    M, N, K = case["M"], case["N"], case["K"]
    return dict(bytes=2 * M * K + N * K * 17 // 32 + 2 * M * N, flops=2 * M * N * K)


# ---- in 64 bits ------------------------------------------------------------------------------

def _exact_quantized(x):
    """The values 4-bit rows stand for, of float64 x."""
    y = x.unflatten(-1, (-1, BLOCK))
    a = y.abs().amax(-1, keepdim=True)
    e = torch.where(a > 0, torch.floor(torch.log2(a)) - 2, -127.0).clamp_min(-127)
    y = y * torch.exp2(-e)
    # codes lie 0.5 apart below 2, 1 apart below 4, 2 apart above
    step = torch.where(y.abs() < 2, 0.5, torch.where(y.abs() < 4, 1.0, 2.0))
    return ((torch.round(y / step) * step).clamp(-6, 6) * torch.exp2(e)).flatten(-2)


def _exact_weight(codes, scales):
    out = torch.empty(codes.shape[0], 2 * codes.shape[1], dtype=torch.float64, device=codes.device)
    for half in (0, 1):
        c = (codes // 16 if half else codes % 16).long()
        man, exp = c % 2, c // 2 % 4
        mag = torch.where(exp > 0, (2.0 + man) * 2.0 ** (exp.double() - 2), 0.5 * man)
        out[:, half::2] = torch.where(c >= 8, -mag, mag)
    return out * torch.exp2(scales.double() - 127).repeat_interleave(BLOCK, -1)


def exact(case, seed):
    st = prepare(case, seed)
    x = st["x"].double()
    if case["kind"] == "quant":
        return _exact_quantized(x)
    if case["kind"] == "norm":
        H = case["H"]
        if case["post"]:
            x = x / torch.sqrt(x.square().sum(-1, keepdim=True) / H + EPS) * st["post"].double()
        if st["gate"] is not None:
            x = x * st["gate"].double()
        r = st["residual"].double() + st["scale"] * x
        return r / torch.sqrt(r.square().sum(-1, keepdim=True) / H + EPS) * st["weight"].double(), r
    if case["kind"] == "both":
        x = _exact_quantized(x)
    return x @ _exact_weight(st["codes"], st["scales"]).t().contiguous()
