"""The attention's sums are in 32 bits: only the weights that meet the values are rounded to the cache's type.

Every logit here is one product of a power of two and a number of the cache's type, so it is exact, and what may be off is small
enough to tell a sum of unrounded weights from one of rounded ones. With s the logits, R their range in a sequence, n its rows:
* a scaled logit has three roundings (log2 e, its product with the scale, the product with the logit): 2^-22 |s|; what a running
  maximum is off by is the same for all of a head's weights. A weight adds a subtraction, 2^-24 of the difference (at most 1.5 R in base
  2), and 2^-22 for 2^x. The ranges are below 8 in base 2, so no maximum is replaced.
* a sum of weights has at most n / 48 + 24 additions one behind the other (a tile's 12 and the lanes' 2, a tile after the other, the
  join's 8): 2^-24 each. So the sum is off by (relative) e = 2^-22 (max |s| + 1) + 1.5 2^-24 R + (n / 48 + 24) 2^-24.
* lse = (m + log2 l) ln 2: 2^-23 of log2 l for the logarithm, 2^-24 of the sum, two roundings with ln 2, the largest number among
  them being 1.5 max(|s|, |lse|): e + 2^-21 (1 + max |s| + |lse|).
* a slot's weight of a head is 2^(s - lse): the logit's error, that of lse, 2^-24 of the difference (1.5 |s - lse|) and 2^-22; heads / 4 + 4
  additions, and one with the score before (0 here).
"""
import math

import pytest
import torch

import amd_developer_challenge_2025_b200 as pkg
from amd_developer_challenge_2025_b200.fp8_mm import check_device_status

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
DV, D = 128, 192
KINDS = ["half way", "spread"]
LENS = [[2049, 300, 48, 0, 1], [190, 64, 1]]


def problem(lens, heads, dtype, kind, device):
    """(rows of every sequence, q, scale)"""
    g = torch.Generator(device=device).manual_seed(heads + len(lens))
    q = torch.zeros(len(lens), heads, D, dtype=TYPES[dtype], device=device)
    element = DV + torch.arange(heads, device=device) % (D - DV)
    rows = [torch.randn(n, D, generator=g, device=device).to(TYPES[dtype]) for n in lens]
    if kind == "half way":
        # One row in 16 has the weight 1, all others one that either type rounds by nearly half a step, and down.
        scale = -math.log(0.75 + 2.0 ** -9 - 2.0 ** -12 - 2.0 ** -16)
        q[:, torch.arange(heads, device=device), element] = 1.0
        for x in rows:
            x[:, DV:] = -1.0
            x[::16, DV:] = 0.0
    else:
        scale = 0.5
        q[:, torch.arange(heads, device=device), element] = torch.where(torch.arange(heads, device=device) % 3 > 0, 1.0, -0.5).to(q.dtype)
        for x in rows:
            x[:, DV:] = (5 * torch.rand(len(x), D - DV, generator=g, device=device)).to(x.dtype)
    return rows, q, float(torch.tensor(scale, dtype=torch.float32))


def check(rows, q, scale, lse, score):
    heads = q.shape[1]
    for i, x in enumerate(rows):
        n = len(x)
        if n == 0:
            assert (lse[i] == -math.inf).all() and (score[i] == 0).all()
            continue
        s = scale * (q[i].double() @ x.double().T)  # [heads, rows]
        want = torch.logsumexp(s, 1)
        p = torch.exp(s - want[:, None])
        most, spread = s.abs().amax(1), s.amax(1) - s.amin(1)
        assert float(spread.max()) < 5.5
        e = 2.0 ** -22 * (most + 1) + 1.5 * 2.0 ** -24 * spread + (n / 48 + 24) * 2.0 ** -24
        off_lse = e + 2.0 ** -21 * (1 + most + want.abs())
        err = (lse[i].double() - want).abs()
        assert (err <= off_lse).all(), ("lse", i, n, float((err / off_lse).max()))
        each = 2.0 ** -22 * (s.abs() + 1) + off_lse[:, None] + 1.5 * 2.0 ** -24 * (s - want[:, None]).abs() + (heads / 4 + 4) * 2.0 ** -24
        tol = (p * each).sum(0)
        err = (score[i, :n].double() - p.sum(0)).abs()
        assert (err <= tol).all(), ("score", i, n, float((err / tol).max()))
        assert abs(float(score[i, :n].double().sum()) - heads) <= float(tol.sum()), ("all slots", i, n)


def in_32_bits(rows, q, scale, round_sum=False, round_score=False):
    """What the formulas give in 32 bits, with the weights rounded to the cache's type before they are summed where asked for."""
    lse = torch.full(q.shape[:2], -math.inf)
    score = torch.zeros(len(rows), max(len(x) for x in rows))
    for i, x in enumerate(rows):
        if len(x) == 0:
            continue
        t = (q[i].float() @ x.float().T) * (torch.tensor(scale) * 1.4426950408889634)
        m = t.amax(1, keepdim=True)
        w = torch.exp2(t - m)
        rounded = w.to(q.dtype).float()
        total = (rounded if round_sum else w).sum(1, keepdim=True)
        lse[i] = ((m + torch.log2(total)) * math.log(2))[:, 0]
        score[i, :len(x)] = (rounded / total if round_score else torch.exp2(t - m - torch.log2(total))).sum(0)
    return lse, score


@pytest.mark.parametrize("lens", LENS, ids=["split", "whole"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", KINDS)
def test_the_tolerances_see_rounded_weights(kind, dtype, lens):
    """Sums in 32 bits pass; with weights of one row's error (the type's half step) in the sum of a head or of a slot, the first kind fails."""
    made = problem(lens, 40, dtype, kind, "cpu")
    check(*made, *in_32_bits(*made))
    if kind == "half way":
        for mistake, where in ((dict(round_sum=True), "lse"), (dict(round_score=True), "score")):
            with pytest.raises(AssertionError, match=where):
                check(*made, *in_32_bits(*made, **mistake))


@pytest.mark.gpu
@pytest.mark.parametrize("lens", LENS, ids=["split", "whole"])
@pytest.mark.parametrize("heads,page", [(3, 16), (16, 5), (32, 48), (40, 16), (128, 64)])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", KINDS)
def test_sums_in_32_bits(kind, dtype, heads, page, lens):
    rows, q, scale = problem(lens, heads, dtype, kind, "cuda")
    per = -(-max(lens) // page)
    table = torch.randperm(len(lens) * per, device="cuda").int().view(len(lens), per)
    cache = torch.zeros(len(lens) * per, page, D, dtype=TYPES[dtype], device="cuda")
    for i, x in enumerate(rows):
        slot = torch.arange(len(x), device="cuda")
        cache[table[i, slot // page].long(), slot % page] = x
    score = torch.zeros(len(lens), per * page, device="cuda")
    lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
    _, lse = pkg.mla_cache_attend(q, cache, table, lens, DV, scale, score=score, max_len=int(lens.max()), return_lse=True)
    check_device_status()
    check(rows, q, scale, lse, score)
