"""Every kernel, tile and split that the plan of a product with 4-bit weights chooses, on whole numbers.

CPU: coopt_mxfp4_linear_plan over sizes drawn from decoding, verify and prompt rows by the widths and lengths
around the models' own finds no way of running a product that the cases below lack.  GPU: each of them
against a product in 64 bits.  |x| <= 12 in steps of 1, |w| <= 12 in steps of 1/4, blocks of different scales on both
sides: sums of K <= 14336 products are multiples of 1/4 below 2^21, exact in fp32 in any order, so the bf16
output is the exact sum rounded once.
"""
import ctypes
import math
import random

import pytest
import torch

import iitj_llm_coopt_amd as M
from iitj_llm_coopt_amd import _lib, fused

# (rows, N, K) by activations and by whether the K slices are left to a consumer
CASES = {
  ("bf16", False): [
    (1, 70, 4096), (2, 75, 3648), (3, 6144, 4096), (7, 6163, 3648), (9, 70, 8192), (9, 2064, 7776),
    (10, 71, 7872), (10, 76, 2560), (11, 4227, 7712), (12, 2060, 8192), (13, 4079, 8192), (17, 73, 2144),
    (17, 74, 2560), (18, 72, 2048), (18, 118, 1536), (23, 94, 1568), (26, 126, 1248), (67, 2731, 4992),
    (74, 2695, 5120), (130, 787, 3104), (130, 796, 3584), (130, 21871, 1120), (162, 1030, 4192),
    (195, 4984, 4704), (226, 1294, 5632), (231, 2068, 1120), (233, 1319, 5152), (236, 795, 4608),
    (267, 1858, 4928), (290, 1627, 1536), (324, 1486, 2048), (366, 2701, 1120), (380, 1348, 5120),
    (449, 2223, 5120), (513, 1942, 2048), (517, 1927, 1536), (573, 4347, 1664), (580, 1777, 6624),
    (621, 1639, 6528), (658, 3724, 2048), (669, 7371, 1952), (708, 2854, 1536), (724, 3239, 1536),
    (758, 1292, 6400), (881, 5456, 1536), (883, 2871, 1120), (915, 5597, 1216), (963, 5089, 2048),
    (1128, 4517, 1664), (1441, 3362, 1696),
  ],
  ("bf16", True): [
    (1, 224, 1312), (5, 128, 2048), (7, 96, 2400), (9, 2048, 1536), (9, 2048, 2048), (9, 2080, 1568),
    (9, 4096, 1536), (9, 4128, 2048), (11, 4096, 1152), (11, 4160, 1568), (14, 2080, 1120), (24, 96, 1536),
    (27, 128, 1216), (65, 3808, 3584), (67, 3616, 3232), (129, 21888, 1536), (129, 23040, 1600),
    (131, 21984, 2048), (161, 928, 2560), (163, 1376, 3584), (197, 1568, 4352), (230, 1088, 3104),
    (230, 2112, 3584), (245, 704, 2112), (281, 1824, 4640), (291, 1632, 1600), (402, 1248, 5120),
    (529, 2464, 4896), (582, 3456, 1152), (583, 1792, 1568), (584, 1728, 5120), (607, 1696, 5056),
    (613, 2240, 4800), (669, 3776, 1152), (734, 3328, 1568), (741, 2880, 1600), (769, 1792, 4736),
    (806, 2464, 2048), (811, 3040, 1536), (851, 6176, 1440), (882, 2720, 2048), (897, 5472, 1120),
    (1049, 4704, 1824), (1457, 3424, 1408),
  ],
  ("mxfp4", False): [
    (1, 70, 4096), (1, 6132, 4096), (1, 6186, 3616), (2, 70, 3872), (9, 71, 4160), (11, 16403, 1120),
    (15, 72, 2240), (17, 75, 3872), (17, 76, 2048), (21, 16561, 3648), (33, 74, 3680), (39, 3098, 1120),
    (66, 70, 1600), (66, 78, 3136), (67, 78, 1152), (100, 2190, 4608), (146, 16624, 1568), (296, 4139, 13824),
    (489, 2795, 12704), (669, 5511, 1600), (769, 18950, 2816), (1173, 10067, 1696), (1175, 6616, 1600),
    (1253, 6934, 1824), (1253, 7022, 2624),
  ],
  ("mxfp4", True): [
    (2, 96, 2880), (5, 128, 2048), (8, 160, 1536), (9, 96, 8352), (9, 2048, 1536), (9, 2048, 2048),
    (9, 4096, 2048), (9, 4128, 1152), (11, 2080, 1120), (12, 4096, 1536), (12, 4128, 1600), (14, 16736, 3680),
    (15, 2048, 1568), (17, 96, 7744), (20, 16576, 1120), (34, 3104, 3616), (35, 96, 1216), (35, 96, 7840),
    (38, 3136, 7776), (38, 22848, 1120), (65, 96, 1120), (99, 8896, 1216), (109, 2336, 3232),
    (116, 8256, 1568), (136, 5536, 12800), (264, 19680, 1600), (386, 33440, 1600), (708, 2016, 12576),
    (918, 5216, 1600), (1155, 3328, 1120), (1166, 6496, 1888), (1285, 15136, 1664), (1287, 8064, 1568),
    (1290, 6048, 1120), (1292, 7488, 2080),
  ],
}
FLAT = [(a, d, s) for (a, d), shapes in CASES.items() for s in shapes]


def way(rows, N, K, activations, deferred):
    """What tells one way of running a product from another: the kernel, its tile, whether K is split and for whom, how
    many tiles (1, 2, more) a block takes, and how K ends: within a quad of 512 or a step of 128, after an even or
    odd number of quads, and after which of a quad's steps where the widest tile skips the rest."""
    plan = (ctypes.c_int * 8)()
    act4 = activations == "mxfp4"
    assert _lib.load().coopt_mxfp4_linear_plan(rows, N, K, act4, deferred, plan) == _lib.COOPT_OK
    tile, form, mt, nt, wm, wn, ks, deep = plan
    tail = form != 1 and K % 512 != 0
    return (tile, form, mt, nt, wm, wn, ks > 1, deferred and ks > 1, min(deep, 3), tail,
            -(-K // 512) % 2 if tile and ks == 1 else None, -(-K // 128) % 4 if tail and tile and mt * nt > 10 else None)


def test_the_cases_reach_every_way():
    reached = {way(*s, a, d) for a, d, s in FLAT}
    rng = random.Random(0)
    log = lambda lo, hi: int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    for _ in range(200000):
        rows, N = rng.choice([log(1, 256), log(1, 4093)]), log(16, 40000)
        K = rng.choice([32 * log(1, 448), 512 * log(1, 28)])
        deferred = rng.random() < 0.5
        if deferred:
            N = max(32, N // 32 * 32)
        activations = rng.choice(["bf16", "mxfp4"])
        assert way(rows, N, K, activations, deferred) in reached, (rows, N, K, activations, deferred)


def test_the_plan_refuses():
    plan = _lib.load().coopt_mxfp4_linear_plan
    assert plan(1, 16, 32, 0, 0, None) == _lib.COOPT_EINVAL
    out = (ctypes.c_int * 8)()
    for bad in ((0, 16, 32), (1, 0, 32), (1, 16, 48), ((1 << 19) + 1, 16, 32)):
        assert plan(*bad, 0, 0, out) == _lib.COOPT_EINVAL and "unsupported" in _lib.last_error()


def operands(dev, rows, N, K):
    """x [rows, K] and the weight [N, K] in float64, and the weight's codes and scales."""
    g = torch.Generator(device=dev).manual_seed(rows + N + K)
    draw = lambda lo, hi, *size: torch.randint(lo, hi, size, generator=g, device=dev, dtype=torch.uint8)
    codes, scales = draw(0, 256, N, K // 2), draw(126, 129, N, K // 32)
    grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=dev)
    grid = torch.cat([grid, -grid])
    w = grid[torch.stack([codes & 15, codes >> 4], -1).flatten(1).int()].view(N, K // 32, 32)
    w = (w * torch.exp2(scales.double() - 127)[..., None]).view(N, K)
    steps = torch.tensor([-6, -4, -3, -2, -1, 0, 1, 2, 3, 4, 6], dtype=torch.float64, device=dev)
    x = steps[draw(0, 11, rows, K).int()].view(rows, K // 32, 32)
    x[..., 0] = 6   # the largest of its block, so that four bits hold every one
    x = (x * (1 + draw(0, 2, rows, K // 32).double())[..., None]).view(rows, K)
    return x, w, codes, scales


@pytest.mark.gpu
@pytest.mark.parametrize("activations,deferred,shape", FLAT)
def test_each_way_is_exact(dev, activations, deferred, shape):
    rows, N, K = shape
    assert K <= 14336 and 4 * K * 144 < 2 ** 24
    x, w, codes, scales = operands(dev, rows, N, K)
    want = torch.matmul(x, w.t().contiguous()).to(torch.bfloat16)
    y = fused.linear(x.to(torch.bfloat16), M.pack_mxfp4_weight(codes, scales, activations), defer_reduce=deferred)
    split = way(rows, N, K, activations, deferred)[7]
    assert isinstance(y, fused.LinearPartials) == split
    assert torch.equal(y.reduce() if split else y, want)
