"""GPU: fused.residual_norm against its definition in 64 bits.

Tolerance: each output is rounded to bf16 once, half a step (2^-8) of the value.  Before that the fp32
statistics and products are off by a relative 2^-17 at most (a mean of H <= 16384 squares summed as 16 terms a
thread, six lane steps and 16 waves: under 40 roundings of 2^-24, half of that in the root; six roundings
of products; the root's own 2 units), which in a sum of residual and branch counts against their magnitudes.
"""
import pytest
import torch

from iitj_llm_coopt_amd import fused

pytestmark = pytest.mark.gpu


def reference(x, residual, weight, eps, post, gate, bs, rs):
    """float64 (out, residual_out) and the magnitudes their errors count against."""
    b = x.double()
    if post is not None:
        b = b / torch.sqrt((b * b).mean(-1, keepdim=True) + eps) * post.double()
    if gate is not None:
        b = b * gate.double()
    r = rs * residual.double() + bs * b
    mag = abs(rs) * residual.double().abs() + abs(bs) * b.abs()
    inv = weight.double() / torch.sqrt((r * r).mean(-1, keepdim=True) + eps)
    return r * inv, r, mag * inv.abs(), mag


def check(got, new, ref):
    out, r, mag_out, mag_r = ref
    assert ((got.double() - out).abs() <= 2.0 ** -8 * out.abs() + 2.0 ** -17 * mag_out).all()
    assert ((new.double() - r).abs() <= 2.0 ** -8 * r.abs() + 2.0 ** -17 * mag_r).all()


def inputs(dev, T, H, gate, post, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed + T + H)
    randn = lambda *s: torch.randn(*s, generator=g, device=dev)
    x, residual = (3 * randn(T, H)).to(torch.bfloat16), (10 * randn(T, H)).to(torch.bfloat16)
    weight, pw = (1 + 0.3 * randn(H)).to(torch.bfloat16), (1 + 0.3 * randn(H)).to(torch.bfloat16)
    gates = {None: None, "channel": randn(H).to(torch.bfloat16), "token": randn(T, H).to(torch.bfloat16)}
    return x, residual, weight, pw if post else None, gates[gate]


@pytest.mark.parametrize("post", [True, False])
@pytest.mark.parametrize("gate", [None, "channel", "token"])
@pytest.mark.parametrize("T,H", [(1, 8), (2, 16), (1, 4096), (3, 504), (5, 512), (7, 520), (160, 2048), (33, 2056), (9, 4096),
                                 (4, 4104), (3, 8192), (2, 8200), (2, 16384), (1, 16376), (4093, 256)])
def test_matches_the_definition(dev, T, H, gate, post):
    x, residual, weight, pw, gv = inputs(dev, T, H, gate, post)
    ref = reference(x, residual, weight, 1e-5, pw, gv, 0.25, 1.5)
    new, before = torch.empty_like(residual), residual.clone()
    got = fused.residual_norm(x, residual, weight, 1e-5, post_weight=pw, gate=gv, branch_scale=0.25,
                              residual_scale=1.5, residual_out=new)
    check(got, new, ref)
    assert torch.equal(residual, before)
    # in place, the default, with the same bits
    out = torch.empty_like(x)
    assert fused.residual_norm(x, residual, weight, 1e-5, pw, gv, 0.25, 1.5, out=out) is out
    assert torch.equal(out, got) and torch.equal(residual, new)


def test_from_partial_sums(dev):
    """x as the unreduced output of a projection: the same bits as from the reduced one."""
    H, K = 1024, 8192
    x = torch.randn(40, K, device=dev).to(torch.bfloat16)
    w = (0.02 * torch.randn(H, K, device=dev)).to(torch.bfloat16)
    _, residual, weight, pw, gv = inputs(dev, 40, H, "token", True)
    part = fused.linear(x, w, defer_reduce=True)
    assert isinstance(part, fused.LinearPartials) and part.ks > 1
    full = part.reduce()
    new = [torch.empty_like(residual) for _ in range(2)]
    got = [fused.residual_norm(h, residual, weight, 1e-6, pw, gv, 0.5, residual_out=n)
           for h, n in zip((part, full), new)]
    assert torch.equal(*got) and torch.equal(*new)
    check(got[0], new[0], reference(full, residual, weight, 1e-6, pw, gv, 0.5, 1.0))


@pytest.mark.parametrize("ks", [1, 3, 4, 5, 8, 9, 16])
@pytest.mark.parametrize("H", [8, 520, 4096, 8192, 16384])
def test_any_number_of_slices(dev, H, ks):
    """1 to 16 slices of partial sums at every block size: the bits of their sum in order, rounded once."""
    T, padded = 5, 16
    x, residual, weight, pw, gv = inputs(dev, T, H, "channel", True)
    buf = torch.randn(ks * padded * H, device=dev)
    part = fused.LinearPartials(buf.view(torch.uint8), ks, T, padded, H, x.shape, x.device)
    want_new = torch.empty_like(residual)
    want = fused.residual_norm(part.reduce(), residual, weight, 1e-6, pw, gv, 0.5, residual_out=want_new)
    got = fused.residual_norm(part, residual, weight, 1e-6, pw, gv, 0.5)
    assert torch.equal(got, want) and torch.equal(residual, want_new)


def test_rows_are_their_own(dev):
    """A row that is not finite, a row of zeros and one of the largest values change no other row."""
    T, H = 6, 640
    x, residual, weight, pw, gv = inputs(dev, T, H, "channel", True)
    base = fused.residual_norm(x, residual, weight, 1e-5, pw, gv, residual_out=torch.empty_like(x))
    x[1, 5], x[2], residual[2] = float("inf"), 0, 0
    x[4] = 3e38
    new = torch.empty_like(x)
    got = fused.residual_norm(x, residual, weight, 1e-5, pw, gv, residual_out=new)
    keep = [0, 3, 5]
    assert torch.equal(got[keep], base[keep])
    assert (got[2] == 0).all() and (new[2] == 0).all()


def test_strides_shapes_and_gates(dev):
    x, residual, weight, pw, gv = inputs(dev, 6, 264, "token", True)
    want = fused.residual_norm(x, residual, weight, 1e-5, pw, gv, residual_out=torch.empty_like(x))
    wide = torch.zeros(6, 400, dtype=torch.bfloat16, device=dev)
    for off in (0, 8):
        wide[:, off:off + 264] = gv
        got = fused.residual_norm(x, residual, weight, 1e-5, pw, wide[:, off:off + 264], residual_out=torch.empty_like(x))
        assert torch.equal(got, want)
    v = lambda t: t.view(2, 3, 264)
    got = fused.residual_norm(v(x), v(residual), weight, 1e-5, pw, v(gv), residual_out=torch.empty_like(v(x)))
    assert torch.equal(got, v(want))
    one = fused.residual_norm(x[:1], residual[:1], weight, 1e-5, pw, gv[:1], residual_out=torch.empty_like(x[:1]))
    assert torch.equal(one, want[:1])
    assert fused.residual_norm(x[:0], residual[:0], weight, 1e-5, pw, gv[:0]).shape == (0, 264)


def test_graph_replays(dev):
    x, residual, weight, pw, gv = inputs(dev, 32, 2048, "channel", True)
    start = residual.clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = fused.residual_norm(x, residual, weight, 1e-5, pw, gv, 0.5)
    for i in range(3):
        x.copy_(torch.randn_like(x))
        residual.copy_(start)
        g.replay()
        new = torch.empty_like(start)
        want = fused.residual_norm(x, start, weight, 1e-5, pw, gv, 0.5, residual_out=new)
        assert torch.equal(out, want) and torch.equal(residual, new), i


def test_more_rows_than_a_launch(dev):
    """Past 2^21 rows the work goes in several launches: the same bits as of the rows alone."""
    T, H = (1 << 21) + 5, 8
    x, residual, weight, pw, gate = inputs(dev, T, H, "token", True)
    new = torch.empty_like(residual)
    got = fused.residual_norm(x, residual, weight, 1e-5, pw, gate, residual_out=new)
    for rows in (slice(0, 100), slice((1 << 21) - 50, None)):
        r = torch.empty_like(residual[rows])
        o = fused.residual_norm(x[rows], residual[rows], weight, 1e-5, pw, gate[rows], residual_out=r)
        assert torch.equal(o, got[rows]) and torch.equal(r, new[rows])


def test_results_over_inputs(dev):
    """out in the place of x, of the residual or of the gate, residual_out in that of x; both in one place are refused."""
    x, residual, weight, pw, gate = inputs(dev, 9, 520, "token", True)
    new = torch.empty_like(residual)
    want = fused.residual_norm(x, residual, weight, 1e-5, pw, gate, residual_out=new)
    for name in ("x", "gate", "residual"):
        a = dict(x=x.clone(), residual=residual.clone(), gate=gate.clone())
        other = torch.empty_like(residual)
        fused.residual_norm(a["x"], a["residual"], weight, 1e-5, pw, a["gate"], residual_out=other, out=a[name])
        assert torch.equal(a[name], want) and torch.equal(other, new)
    a = x.clone()
    assert torch.equal(fused.residual_norm(a, residual, weight, 1e-5, pw, gate, residual_out=a), want)
    assert torch.equal(a, new)
    before = residual.clone()
    with pytest.raises(ValueError, match="same rows"):
        fused.residual_norm(x, residual, weight, 1e-5, pw, gate, out=residual)
    with pytest.raises(ValueError, match="16384"):
        wide = torch.zeros(1, 16392, device=dev, dtype=torch.bfloat16)
        fused.residual_norm(wide, wide.clone(), wide[0], 1e-5)
    assert torch.equal(residual, before)
