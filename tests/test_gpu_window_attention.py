"""GPU: paged attention with a sliding window and first tokens that stay visible, and over 4-bit
caches, against the closed form in float64.

Tolerance, per output element, from the roundings the operator is allowed:
  |out - ref| <= u |ref|                        the bf16 output, u = 2^-8
              + (u_p + 2 ds + 2^-18) A          A = sum_k w_k |v_k| of the row
u_p: a probability rounded to 16 bits next to its value (bf16 caches 2^-8; codes 2^-11, fp16);
an INT8 value of the definition is itself rounded to bf16, which the kernel need not do (2^-8).
ds: the error of a score: a product of D terms summed in fp32 in any order, D 2^-24 sum |q||k|,
where a 4-bit key enters as code plus 8 (|k| + 24 s covers it), and 2^-22 of the score for the
exponent.  Beside 4-bit keys q is the sum of two 4-bit numbers: its elements under 2^-9 of the row's
largest are rounded to steps of 2^-17 of it, 2^-18 max|q| sum |k| at most.
Both numerator and sum move by ds (2 ds).  2^-18 A covers the fp32 sums over up to 2^6 tiles, each
a rounding of 2^-24 of the magnitudes summed so far.  A 4-bit value is summed as code plus 8, and 8
times the sum of w s is taken off at the end: the magnitudes summed are |v| + 8 s, not |v| alone, so
there the last term is 2^-18 sum_k w_k (|v_k| + 8 s_k).  (Where every code of an element is 0, |v| is
0 and these roundings, up to 64 * 2^-24 * 8 s, are all of the error.)  Its operand is a subnormal
number of the matrix cores, whose products keep 2^-20 of the largest: four such tiles make 2^-18.

Codes again: the probabilities times the values' scales, P' = p s 2^-e in fp16, have steps of 2^-24
below 2^-14 and are off by up to 2^-25 there, whatever they are themselves.  2^e <= 2^-6 S, S the
sequence's largest scale, and p is 2^(score - r) with a reference r that one of the row's scores
had, so sum p >= 1 and the output moves by at most 2^-25 2^e sum |c| / sum p <= 2^-31 S sum |c| over the
codes c the row sees.  (Only where the row's heavy keys have codes of 0 is this not hidden by the
terms above: one key with nearly all the weight and a 0 there leaves A the size of the light keys'.)
"""
import numpy as np
import pytest
import torch

import iitj_llm_coopt_amd as M
from iitj_llm_coopt_amd import _lib
from oracle import codec as OC

pytestmark = pytest.mark.gpu


def closed_form(q, K, V, scale, window, sinks, kv, s_k, s_v):
    """float64 (out, tol) of one sequence: q [n, Hq, D], K / V [L, Hkv, D], their scales s_k, s_v
    [L, Hkv] (None for bf16)."""
    n, Hq, D = q.shape
    L, Hkv, _ = K.shape
    out, tol = np.zeros((n, Hq, D)), np.zeros((n, Hq, D))
    k = np.arange(L)
    for j in range(n):
        p = L - n + j
        see = k <= p
        if window is not None:
            see &= (k > p - window) | (k < sinks)
        if not see.any():
            continue
        for h in range(Hq):
            g = h // (Hq // Hkv)
            Ks, Vs = K[see, g], V[see, g]
            s = Ks @ q[j, h] * scale
            w = np.exp(s - s.max())
            w /= w.sum()
            out[j, h] = w @ Vs
            mag = np.abs(Ks) @ np.abs(q[j, h])
            if kv == "int4":
                mag = mag + 24 * s_k[see, g] * np.abs(q[j, h]).sum()
            ds = (D * 2.0 ** -24 * mag * scale).max() + 2.0 ** -22 * np.abs(s).max()
            if kv == "int4":
                ds += 2.0 ** -18 * np.abs(q[j, h]).max() * np.abs(Ks).sum(1).max() * scale
            u_p = {"auto": 2.0 ** -8, "int8": 2.0 ** -11 + 2.0 ** -8, "int4": 2.0 ** -11}[kv]
            A = w @ np.abs(Vs)
            summed = A + (8 * (w @ s_v[see, g]) if kv == "int4" else 0)
            tol[j, h] = 2.0 ** -8 * np.abs(out[j, h]) + (u_p + 2 * ds) * A + 2.0 ** -18 * summed
            if kv != "auto":
                codes = (np.abs(Vs) / np.maximum(s_v[see, g], 1e-30)[:, None]).sum(0)
                tol[j, h] += 2.0 ** -31 * s_v[:, g].max() * codes
    return out, tol


class Setup:
    """Sequences (rows, keys) over a pool of scattered pages.  Every place no row may see holds NaN
    (bf16 values, scales): pages of no sequence, keys past a sequence's end, keys below all windows
    (whose table entries are also out of the pool)."""

    def __init__(self, dev, seqs, Hq, Hkv, D, kv, window=None, sinks=0, bs=16, layout="head", seed=0,
                 poison=True, magnitude=1.0, outlier=0.0):
        self.dev, self.seqs, self.kv, self.D, self.window, self.sinks, self.bs = dev, seqs, kv, D, window, sinks, bs
        rng = np.random.default_rng(seed)
        widths = [-(-L // bs) for _, L in seqs]
        nb = sum(widths) + 3
        perm = rng.permutation(nb)
        self.table_np = np.full((len(seqs), max(max(widths), 1) + 1), -7, np.int32)
        self.K, self.V, self.sk, self.sv = [], [], [], []
        store = {"head": (nb, Hkv, bs, D), "token": (nb, bs, Hkv, D), "padded": (nb, bs + 1, Hkv + 2, D + 32)}[layout]

        def view(t, last):
            if layout == "head":
                return t.transpose(1, 2)
            return t if layout == "token" else t[:, :bs, :Hkv, :last]

        if kv == "auto":
            full = [torch.full(store, float("nan") if poison else 0.0, dtype=torch.bfloat16) for _ in range(2)]
            self.caches, self.scales = [view(t, D) for t in full], [None, None]
        else:
            cstore = store if kv == "int8" else (*store[:3], store[3] // 2)
            dt = torch.int8 if kv == "int8" else torch.uint8
            full = [torch.from_numpy(rng.integers(-127, 128, cstore).astype(np.int8)).view(dt) for _ in range(2)]
            sc = [torch.full(store[:3], float("nan") if poison else 0.0, dtype=torch.float16) for _ in range(2)]
            self.caches = [view(t, D if kv == "int8" else D // 2) for t in full]
            self.scales = [view(t.unsqueeze(-1), 1).squeeze(-1) for t in sc]
        o = 0
        for b, (n, L) in enumerate(seqs):
            pages = perm[o:o + widths[b]]
            o += widths[b]
            self.table_np[b, : widths[b]] = pages
            x = rng.standard_normal((2, L, Hkv, D)) * magnitude
            if outlier:
                x = np.where(rng.random(x.shape) < outlier, 20 * x, x)
            x = x.astype(np.float32)
            vals = []
            first = L - n - (window or 1 << 30) + 1       # keys [sinks, first) are seen by no row
            hidden = np.arange(L)
            hidden = (hidden >= sinks) & (hidden < first)
            for i in range(2):
                blk, off = torch.from_numpy(pages[np.arange(L) // bs].astype(np.int64)), torch.arange(L) % bs
                if kv == "auto":
                    y = torch.from_numpy(x[i]).to(torch.bfloat16)
                    vals.append(y.double().numpy())
                    if poison:
                        y[torch.from_numpy(hidden)] = float("nan")
                    self.caches[i][blk, off] = y
                else:
                    c, s = OC.quantize(x[i], 8 if kv == "int8" else 4)
                    v = OC_values(c, s, kv)
                    vals.append(v)
                    s = torch.from_numpy(np.asarray(s, np.float16))
                    (self.sk, self.sv)[i].append(s.double().numpy())
                    if poison:
                        s[torch.from_numpy(hidden)] = float("nan")
                    self.caches[i][blk, off] = torch.from_numpy(c)
                    self.scales[i][blk, off] = s
            if poison:
                for w in range(widths[b]):
                    if hidden[w * bs:(w + 1) * bs].all() and (w + 1) * bs <= L:
                        self.table_np[b, w] = [-1, nb + 5, 2 ** 31 - 1][w % 3]
            self.K.append(vals[0])
            self.V.append(vals[1])
            if kv == "auto":
                self.sk.append(None)
                self.sv.append(None)

        def move(t):     # to the GPU with its strides
            if t is None:
                return None
            base = t if t._base is None else t._base
            while base._base is not None:
                base = base._base
            return torch.as_strided(base.to(dev), t.shape, t.stride(), t.storage_offset())

        self.caches, self.scales = [move(t) for t in self.caches], [move(t) for t in self.scales]
        self.table = torch.from_numpy(self.table_np).to(dev)
        rows = [n for n, _ in seqs]
        self.cu = torch.tensor(np.concatenate([[0], np.cumsum(rows)]), dtype=torch.int32, device=dev)
        self.lens = torch.tensor([L for _, L in seqs], dtype=torch.int32, device=dev)
        self.T, self.max_q, self.max_k = sum(rows), max(max(rows), 1), max(max(L for _, L in seqs), 1)
        self.q = torch.from_numpy(rng.standard_normal((self.T + 2, Hq, D)).astype(np.float32)).to(torch.bfloat16).to(dev)

    def run(self, **kw):
        """The call, with two rows behind the last sequence that must stay as they are."""
        out = torch.full_like(self.q, 7.0)
        kw = dict(dict(window=self.window, sink_tokens=self.sinks, out=out), **kw)
        got = M.flash_attn_varlen_func(
            q=self.q, k=self.caches[0], v=self.caches[1], cu_seqlens_q=self.cu, max_seqlen_q=self.max_q,
            seqused_k=self.lens, max_seqlen_k=self.max_k, softmax_scale=self.D ** -0.5, causal=True,
            block_table=self.table, k_scale=self.scales[0], v_scale=self.scales[1], **kw)
        return got

    def check(self, out, note=""):
        o = out.float().cpu().numpy().astype(np.float64)
        q = self.q.double().cpu().numpy()
        assert (o[self.T:] == 7.0).all(), "rows behind the last sequence were written"
        row, worst = 0, 0.0
        for b, (n, L) in enumerate(self.seqs):
            ref, tol = closed_form(q[row:row + n], self.K[b], self.V[b], self.D ** -0.5, self.window,
                                   self.sinks, self.kv, self.sk[b], self.sv[b])
            d = np.abs(o[row:row + n] - ref)
            assert np.isfinite(o[row:row + n]).all(), f"{note} sequence {b}: not finite"
            if d.size:
                worst = max(worst, float((d / np.maximum(tol, 1e-30)).max()) if (tol > 0).any() else 0.0)
                assert (d <= tol).all(), f"{note} sequence {b} (rows {n}, keys {L}): {float((d - tol).max())} over"
            row += n
        print(f"[window] {note} kv={self.kv} D={self.D} window={self.window} sinks={self.sinks}: "
              f"{worst:.2f} of the tolerance", flush=True)


def OC_values(c, s, kv):
    """float64 values the codes stand for: INT8 bf16(code * scale), INT4 code * scale."""
    s = np.asarray(s, np.float16).astype(np.float64)[..., None]
    if kv == "int8":
        return (torch.from_numpy(c.astype(np.float64) * s).to(torch.bfloat16)).double().numpy()
    n = np.stack([(c & 15).astype(np.int64) - 8, (c >> 4).astype(np.int64) - 8], -1).reshape(*c.shape[:-1], 2 * c.shape[-1])
    return n * s


KINDS = ["auto", "int8", "int4"]


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("kv", KINDS)
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 4), (33, 0), (100, 17), (200, 64), (700, 3), (5000, 4),
                                          (31, 32), (64, 300)])
def test_windows_at_decode_and_verify_rows(dev, kv, D, window, sinks):
    """1 to 5 rows, contexts from one key to several hundred, every alignment of the window's edges."""
    seqs = [(1, 1), (1, 2), (5, 5), (3, 31), (1, 32), (2, 33), (5, 100), (1, 257), (4, 300), (5, 611), (0, 40), (1, 48)]
    s = Setup(dev, seqs, 8, 2, D, kv, window, sinks, seed=window + sinks)
    s.check(s.run(), "verify")


@pytest.mark.parametrize("kv", KINDS)
@pytest.mark.parametrize("n", [1, 2, 3, 5, 8, 13, 16])
def test_windows_over_row_counts_of_one_tile_to_four(dev, kv, n):
    """4 query heads a KV head, 4 to 64 rows of it in one block; 7 heads: rows that fill no tile."""
    for Hq, Hkv in ((8, 2), (7, 1)):
        if Hq // Hkv * n > 64:
            continue
        s = Setup(dev, [(n, 150), (n, 700), (max(n - 1, 0), 333)], Hq, Hkv, 128, kv, 130, 5, seed=n)
        s.check(s.run(), f"{n} rows, {Hq}/{Hkv} heads")


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("kv", KINDS)
@pytest.mark.parametrize("window,sinks", [(1, 0), (40, 4), (64, 64), (150, 0), (1000, 8)])
def test_windows_over_chunks(dev, kv, D, window, sinks):
    """Prefill chunks whole and continued, beside verify items and an empty one."""
    seqs = [(257, 257), (100, 400), (5, 333), (1, 90), (0, 10), (65, 65), (17, 600)]
    s = Setup(dev, seqs, 8, 2, D, kv, window, sinks, seed=window)
    s.check(s.run(), "chunks")


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("rows,Hq,Hkv", [(1, 32, 8), (5, 32, 8), (9, 28, 4), (3, 4, 4), (40, 8, 2), (200, 14, 2)])
def test_int4_caches_without_a_window(dev, rows, Hq, Hkv, D):
    s = Setup(dev, [(rows, max(rows, 333)), (max(rows - 1, 1), 517 + rows), (1, 1), (min(rows, 5), 64)], Hq, Hkv, D,
              "int4", seed=rows, outlier=0.01)
    s.check(s.run(), f"int4 {rows} rows")


@pytest.mark.parametrize("kv", KINDS)
@pytest.mark.parametrize("layout", ["token", "padded"])
@pytest.mark.parametrize("bs", [16, 64])
def test_layouts_and_block_sizes(dev, kv, layout, bs):
    for seqs in ([(5, 300), (2, 77)], [(60, 300), (2, 77)]):
        s = Setup(dev, seqs, 8, 4, 128, kv, 100, 4, bs=bs, layout=layout, seed=bs)
        s.check(s.run(), f"{layout} {bs}")
    s = Setup(dev, [(5, 300), (2, 77)], 8, 4, 64, kv, 100, 4, bs=bs, layout=layout, seed=bs)
    s.check(s.run(), f"{layout} {bs}")


@pytest.mark.parametrize("kv,window,sinks,L", [(kv, *w) for kv in KINDS for w in ((1024, 4, 6001), (3000, 100, 9000))] +
                         [("int4", None, 0, 5000)])
def test_long_contexts_are_split_and_joined(dev, kv, window, sinks, L):
    """One sequence of few KV heads: the visible keys are spread over blocks and merged."""
    for D in (64, 128):
        s = Setup(dev, [(1, L), (4, L - 777)], 8, 2, D, kv, window, sinks, seed=L)
        s.check(s.run(), "split")


@pytest.mark.parametrize("kv", KINDS)
def test_rows_that_see_nothing_are_zero(dev, kv):
    """A sequence with fewer keys than rows (its first rows stand before the first key), and none."""
    s = Setup(dev, [(5, 2), (3, 0), (40, 7), (1, 20)], 8, 2, 128, kv, 4, 2)
    out = s.run()
    s.check(out, "empty rows")
    o = out.float().cpu().numpy()
    assert (o[:3] == 0).all() and (o[5:8] == 0).all() and (o[8:41] == 0).all()


@pytest.mark.parametrize("rows,Hq,Hkv", [(4, 8, 2), (40, 8, 2), (300, 64, 8)])
def test_infinities_and_nan_reach_only_the_rows_that_see_them(dev, rows, Hq, Hkv):
    """bf16 keys and values of partly visible positions: rows before them, and rows whose window
    has passed them, are as if the values were finite."""
    L = max(200, rows + 100)
    s = Setup(dev, [(rows, L)], Hq, Hkv, 128, "auto", 50, 3, seed=3)
    clean = s.run().clone()
    first = L - rows
    places = [(0, first + 1, float("nan")), (1, first + 2, float("inf")), (1, first - 49, float("nan")),
              (1, first - 48, float("-inf")), (0, first - 47, float("inf"))]
    for which, key, value in places:
        page, off = int(s.table[0, key // 16]), key % 16
        kept = s.caches[which][page, off].clone()
        s.caches[which][page, off] = value
        got = s.run()
        s.caches[which][page, off] = kept
        for j in range(rows):
            p = first + j
            sees = key <= p and (key > p - 50 or key < 3)
            same = torch.equal(got[j], clean[j])
            assert same or sees, (which, key, value, j)
            if sees and which == 1:
                g = got[j].float()
                assert not torch.isfinite(g).any(), (which, key, value, j)
                assert torch.isnan(g).all() if value != value else (g == value).all()


def takes_staged_kernel(s, Hq, Hkv):
    """Whether the call's windows fill the GPU: 128 rows a window, staged for four waves."""
    most = min(s.max_q, 128) + (s.window or s.max_k) + s.sinks + 128
    return _lib.load().coopt_verify_attention_window_rows(
        _lib.DT_BF16 if s.kv == "auto" else _lib.DT_I8, len(s.seqs), Hq, Hkv, s.D, s.max_q, min(most, s.max_k), s.T) == 128


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("kv,window,sinks", [(kv, *w) for kv in KINDS for w in ((40, 4), (130, 70), (1000, 8))] +
                         [("int4", None, 0)])
def test_batches_that_fill_the_gpu(dev, kv, window, sinks, D):
    """Chunks whole and continued beside short items, 64 query heads: the windows of 128 rows, among
    them some of at most 64 rows, an empty one, and rows before the first key."""
    s = Setup(dev, [(300, 300), (37, 400), (5, 333), (0, 10), (130, 131), (3, 1)], 64, 8, D, kv, window, sinks,
              seed=sinks, outlier=0.01)
    assert takes_staged_kernel(s, 64, 8)
    s.check(s.run(), "full")


@pytest.mark.parametrize("kv", KINDS)
def test_batches_of_more_sequences_than_a_wave(dev, kv):
    """More than 64 sequences: blocks in grid order, short items alone and beside a chunk."""
    short = [(1 + b % 2, 1 + 17 * b % 200) for b in range(70)]
    s = Setup(dev, short, 8, 2, 64, kv, 60, 3, seed=8)
    s.check(s.run(), "70 short")
    s = Setup(dev, [(270, 290)] + [(1, 1 + 17 * b % 200) for b in range(69)], 64, 8, 64, kv, 60, 3, seed=9)
    assert takes_staged_kernel(s, 64, 8)
    s.check(s.run(), "70 with a chunk")


@pytest.mark.parametrize("kv", KINDS)
def test_scores_that_climb_over_the_keys(dev, kv):
    """Each tile's scores lie further above the ones before it, or below: the reference of a row's
    exponents moves at every tile, by more and by less than it may lag behind, or never again."""
    for seqs, Hq, Hkv in (([(3, 700), (1, 90)], 8, 2), ([(300, 420), (2, 64)], 64, 8)):
        for climb in (0.02, 0.3, -0.3):
            s = Setup(dev, seqs, Hq, Hkv, 128, kv, 350, 8, seed=12)
            for b, (n, L) in enumerate(seqs):      # keys along the queries' common direction
                scale = (climb * np.arange(L)).astype(np.float32)
                d = np.ones((Hkv, 128), np.float32) / 8
                x = s.K[b].astype(np.float32) * 0.05 + scale[:, None, None] * d
                blk = torch.from_numpy(s.table_np[b, np.arange(L) // 16].astype(np.int64))
                ok, off = (blk >= 0) & (blk < s.caches[0].shape[0]), torch.arange(L) % 16
                if kv == "auto":
                    y = torch.from_numpy(x).to(torch.bfloat16)
                    s.K[b] = y.double().numpy()
                    s.caches[0][blk[ok].to(dev), off[ok].to(dev)] = y[ok].to(dev)
                else:
                    c, sc = OC.quantize(x, 8 if kv == "int8" else 4)
                    s.K[b], s.sk[b] = OC_values(c, sc, kv), np.asarray(sc, np.float16).astype(np.float64)
                    s.caches[0][blk[ok].to(dev), off[ok].to(dev)] = torch.from_numpy(c)[ok].to(dev)
                    s.scales[0][blk[ok].to(dev), off[ok].to(dev)] = torch.from_numpy(np.asarray(sc, np.float16))[ok].to(dev)
            s.q.mul_(0.1).add_(1.0)
            s.check(s.run(), f"climb {climb} {seqs[0][0]} rows")


@pytest.mark.parametrize("kv", KINDS)
@pytest.mark.parametrize("rows,Hq,Hkv", [(3, 8, 2), (40, 8, 2), (300, 64, 8)])
def test_a_row_that_is_not_finite_is_its_own(dev, kv, rows, Hq, Hkv):
    """A query with a NaN or an infinity among its elements: NaN, and every other row as before (the
    rows of a block share the moments at which references move, so not to the bit)."""
    s = Setup(dev, [(rows, rows + 100)], Hq, Hkv, 128, kv, 90, 4, seed=31)
    clean = s.run().clone()
    for value in (float("nan"), float("inf"), float("-inf")):
        kept = s.q.clone()
        s.q[rows // 2, 1, 5] = value
        got = s.run()
        s.q.copy_(kept)
        assert torch.isnan(got[rows // 2, 1].float()).all(), value
        got[rows // 2, 1] = clean[rows // 2, 1]
        s.check(got, f"beside {value}")


def test_two_threads_on_one_stream(dev):
    """Calls whose parts go through the stream's shared workspace, from two threads at once."""
    import threading
    sets = [Setup(dev, [(2, 5000 + 37 * i)], 8, 2, 128, "int4", None, 0, seed=20 + i) for i in range(2)]
    want = [s.run().clone() for s in sets]
    torch.cuda.synchronize(dev)
    bad = []

    def work(i):
        for _ in range(200):
            if not torch.equal(sets[i].run(), want[i]):
                bad.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad, f"{len(bad)} of 400 calls"


@pytest.mark.parametrize("kv", KINDS)
def test_scores_far_apart_and_large_scales(dev, kv):
    """Outliers 20 times as large, and values of magnitude 1000: maxima that move between tiles."""
    for mag, out in ((1.0, 0.02), (1000.0, 0.0), (1e-3, 0.0)):
        s = Setup(dev, [(3, 700), (1, 90)], 8, 2, 128, kv, 400, 8, magnitude=mag, outlier=out, seed=5)
        if mag == 1000.0:     # keep scores in range: only the values are large
            s.q.mul_(1e-3)
        s.check(s.run(), f"magnitude {mag}")


@pytest.mark.parametrize("kv", KINDS)
@pytest.mark.parametrize("magnitude", [0.0, 1e-30, 1e6])
def test_queries_of_any_magnitude(dev, kv, magnitude):
    """Queries of zeros (every visible key weighs the same), of tiny numbers, and so large that one
    key takes all the weight (scores up to 10^7; the call takes them below 2^30, where the rounded
    maximum of a row is still within a softmax exponent of the score itself)."""
    for seqs in ([(2, 300), (1, 40)], [(50, 300)]):
        s = Setup(dev, seqs, 8, 2, 128, kv, 100, 4, seed=6)
        s.q.mul_(magnitude)
        if magnitude < 1:
            s.check(s.run(), f"queries times {magnitude}")
            continue
        # scores of 1e7: the largest one's value, half a bf16 step off (4-bit and INT8 values are
        # code * scale, INT8's rounded to bf16 in the definition only: one more half step)
        out, row = s.run().double().cpu().numpy(), 0
        q = s.q.double().cpu().numpy()
        for b, (n, L) in enumerate(seqs):
            for j in range(n):
                p, k = L - n + j, np.arange(L)
                see = (k <= p) & ((k > p - 100) | (k < 4))
                for h in range(8):
                    score = np.where(see, s.K[b][:, h // 4] @ q[row, h], -np.inf)
                    best = np.sort(score)[-2:]
                    if best[1] - best[0] < 1e-5 * np.abs(best).max():
                        continue     # a tie within the scores' own error
                    want = s.V[b][score.argmax(), h // 4]
                    assert (np.abs(out[row, h] - want) <= 2.0 ** -7 * np.abs(want) + 2.0 ** -18 * 8 * np.abs(want).max()).all()
                row += 1


@pytest.mark.parametrize("kv", KINDS)
def test_graph_replays_match_eager_calls(dev, kv):
    """Captured once and replayed with new queries, eager work between the replays; twice the same
    bits.  Another stream than the default one."""
    s = Setup(dev, [(1, 4000), (2, 3100)], 8, 2, 128, kv, 2000, 4, seed=9)
    s.run()
    out = torch.full_like(s.q, 7.0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        s.run(out=out)
    gen = torch.Generator(device=dev).manual_seed(1)
    for i in range(4):
        s.q.copy_(torch.randn(s.q.shape, generator=gen, device=dev))
        graph.replay()
        eager = s.run()
        torch.cuda.synchronize()
        assert torch.equal(out, eager), i
        s.check(out, f"replay {i}")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = s.run()
    side.synchronize()
    assert torch.equal(again, eager)


def test_two_graphs_of_one_stream_may_replay_at_once(dev):
    """Each graph holds a workspace of its own: split calls replayed on two streams at once."""
    a = Setup(dev, [(1, 9000)], 8, 2, 128, "int4", seed=1)
    b = Setup(dev, [(2, 8000)], 8, 2, 128, "int4", seed=2)
    outs, graphs = [], []
    for s in (a, b):
        s.run()
        out = torch.full_like(s.q, 7.0)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            s.run(out=out)
        outs.append(out)
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(10):
        for st, g in zip(streams, graphs):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        a.check(outs[0], "graph a")
        b.check(outs[1], "graph b")


def test_pages_past_two_to_the_32_bytes(dev):
    """A bf16 pool of 9 GB, pages at its end."""
    Hkv, D, bs = 8, 128, 16
    nb = 280000                      # 32 KB a page
    kc = torch.empty(nb, Hkv, bs, D, dtype=torch.bfloat16, device=dev).transpose(1, 2)
    small = Setup(dev, [(3, 100)], 16, Hkv, D, "auto", 50, 4, seed=8)
    vc = torch.empty_like(kc)
    w = -(-100 // bs)
    src = small.table[0, :w].clone()
    keep = (src >= 0) & (src < small.caches[0].shape[0])
    dst = torch.arange(nb - w, nb, device=dev, dtype=torch.int32)
    for c, o in ((kc, small.caches[0]), (vc, small.caches[1])):
        c[dst[keep].long()] = o[src[keep].long()]
    want = small.run().clone()
    small.caches = [kc, vc]
    small.table[0, :w] = torch.where(keep, dst, src)
    assert torch.equal(small.run(), want)


def test_the_whole_context_in_the_window_is_plain_attention(dev):
    """bf16: a window as long as the context against the call without one, which other kernels may
    take; both lie within the tolerance of the closed form."""
    s = Setup(dev, [(5, 500), (1, 77), (90, 90)], 8, 2, 128, "auto", None, 0, poison=False)
    s.check(s.run(window=500, sink_tokens=3), "whole")
    s.check(s.run(window=2 ** 40, sink_tokens=2 ** 40), "whole")
    s.check(s.run(window=None, sink_tokens=0), "none")


def test_refusals(dev):
    s = Setup(dev, [(1, 40)], 8, 2, 128, "int4", 10, 0)
    for kw, what in ((dict(window=0), "at least 1"), (dict(window=-3), "at least 1"),
                     (dict(sink_tokens=-1), "negative"), (dict(window=None, sink_tokens=2), "needs a window"),
                     (dict(out=torch.empty(3, 8, 128, device=dev)), "out must be bf16"),
                     (dict(workspace=torch.empty(8, dtype=torch.uint8, device=dev)), "workspace")):
        with pytest.raises(ValueError, match=what):
            s.run(**kw)
    with pytest.raises(TypeError):
        s.run(window=2.5)
    keep = s.scales
    s.scales = [None, None]
    with pytest.raises(ValueError, match="INT4 caches need"):
        s.run()
    s.scales = [keep[0].float(), keep[1].float()]
    with pytest.raises(ValueError, match="fp16"):
        s.run()
    s.scales = keep
    s.table = s.table[:, :2]
    with pytest.raises(ValueError, match="block_table holds"):
        s.run()
    with pytest.raises(ValueError, match="not supported|int4|'auto' or 'int8'"):
        M.paged_attention_qkv(torch.zeros(1, 12 * 128, dtype=torch.bfloat16, device=dev),
                              torch.zeros(1, dtype=torch.int64, device=dev),
                              *(torch.zeros(4, 64, dtype=torch.bfloat16, device=dev) for _ in range(2)),
                              torch.zeros(1, dtype=torch.int64, device=dev),
                              *M.allocate_kv_cache(4, 16, 2, 128, "auto", device=dev)[:2], s.cu, s.lens,
                              torch.zeros(1, 4, dtype=torch.int32, device=dev), 1, 40, 8, kv_cache_dtype="int4")
    assert isinstance(_lib.last_error(), str)
