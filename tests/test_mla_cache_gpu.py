"""The paged-cache operators against plain 64-bit forms.

Tolerances. u is half a step of the type (2^-8 bf16, 2^-11 fp16), A = sum_j p_j |v_j|.
attend: the weights are rounded once (u A), so is the result (u |out|). A logit is a sum of d products in 32 bits, each step off by
at most 2^-23 of the running magnitude (the tensor core truncates): ds = scale * (d + 2) * 2^-23 * max_j sum_i |q_i x_ji|. An error of
ds in every logit moves a normalised weight by a factor of up to exp(2 ds). Exponential, logarithm, scaling and the joins add at
most 2^-20 relative. lse moves by ds + 2^-20 (1 + |lse|), a slot's score by sum_h p_h (2 ds_h + 2^-20) + 2^-22 of the result,
and by 2^-126 a head: below that a 32-bit number is subnormal, spaced 2^-149 or taken for zero, so the relative bounds end there (a
weight of 7e-46 lies between 0 and the smallest subnormal, 1.4e-45).
append: u |y| for the rounding and 2^-20 (|x1| + |x2|) for cosine, sine, products and sum in 32 bits.
evict moves values and compares them: equal."""
import math

import pytest
import torch

import amd_developer_challenge_2025_b200 as pkg
from amd_developer_challenge_2025_b200.fp8_mm import check_device_status

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
NAN = float("nan")


def half_step(t):
    return torch.finfo(t).eps / 2


class Batch:
    """A cache whose pages lie anywhere, NaN wherever no sequence has a row, nonsense in the table behind the last page."""

    def __init__(self, lens, heads, dv=512, dr=64, page=64, dtype="bf16", seed=0, spare=0, cache=None):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.lens_list, self.dv, self.d, self.page, self.dtype = list(lens), dv, dv + dr, page, TYPES[dtype]
        b = len(lens)
        per = (max(lens) + spare) // page + 1
        used = [-(-n // page) for n in lens]
        pages = b * per + 3
        perm = torch.randperm(pages, generator=g, device="cuda")
        if cache is None:
            cache = torch.empty(pages, page, self.d, dtype=self.dtype, device="cuda")
        self.cache = cache.fill_(NAN)
        self.table = torch.full((b, per), -7, dtype=torch.int32, device="cuda")
        self.table[::2] = 1 << 30
        self.rows = []
        for i, n in enumerate(lens):
            ids = perm[i * per:i * per + used[i] + -(-spare // page)]
            self.table[i, :len(ids)] = ids.int()[:per]
            x = torch.randn(n, self.d, generator=g, device="cuda").to(self.dtype)
            slot = torch.arange(n, device="cuda")
            self.cache[ids[slot // page], slot % page] = x
            self.rows.append(x)
        self.lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
        self.q = torch.randn(b, heads, self.d, generator=g, device="cuda").to(self.dtype)
        self.scale = 1 / math.sqrt(128 + dr)
        self.capacity = per * page
        self.g = g

    def attend(self, **more):
        r = pkg.mla_cache_attend(self.q, self.cache, self.table, self.lens, self.dv, self.scale, **more)
        check_device_status()
        return r

    def slots(self, fill=0.0, dtype=torch.float32):
        return torch.full((len(self.rows), self.capacity), fill, dtype=dtype, device="cuda")


def check_attend(bt, out, lse=None, score=None, score0=None):
    for i, x in enumerate(bt.rows):
        n = len(x)
        if n == 0:
            assert (out[i] == 0).all() and (lse is None or (lse[i] == -math.inf).all())
            if score is not None:
                assert torch.equal(score[i], score0[i])
            continue
        x, q = x.double(), bt.q[i].double()
        s = bt.scale * (q @ x.T)
        ds = abs(bt.scale) * (bt.d + 2) * 2.0 ** -23 * (q.abs() @ x.abs().T).amax(1)  # [heads]
        want_lse = torch.logsumexp(s, 1)
        p = torch.exp(s - want_lse[:, None])
        want = p @ x[:, :bt.dv]
        mass = p @ x[:, :bt.dv].abs()
        u = half_step(bt.dtype)
        tol = u * (1 + u) * mass + u * want.abs() + mass * (2 * ds[:, None] + 2.0 ** -20) + 1e-7 * (bt.dtype == torch.float16)
        err = (out[i].double() - want).abs()
        assert (err <= tol).all(), (i, n, float((err / tol).max()))
        if lse is not None:
            assert ((lse[i].double() - want_lse).abs() <= ds + 2.0 ** -20 * (1 + want_lse.abs())).all(), (i, n)
        if score is not None:
            w = score0[i, :n].double() + p.sum(0)
            tol = (p * (2 * ds[:, None] + 2.0 ** -20)).sum(0) + 2.0 ** -22 * w.abs() + len(p) * 2.0 ** -126
            err = (score[i, :n].double() - w).abs()
            assert (err <= tol).all(), (i, n, float((err / tol).max()))
            assert torch.equal(score[i, n:], score0[i, n:])


@pytest.mark.parametrize("heads", [1, 8, 16, 17, 32, 40, 64, 65, 128, 130])
def test_attend_heads(heads):
    bt = Batch([300, 0, 1, 64, 65, 1000], heads, seed=heads)
    check_attend(bt, *bt.attend(return_lse=True))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dv,dr", [(512, 64), (512, 0), (384, 64), (384, 192), (256, 64), (128, 0), (128, 128), (128, 448)])
def test_attend_widths(dv, dr, dtype):
    bt = Batch([129, 777], 20, dv, dr, 32, dtype, seed=dv + dr)
    check_attend(bt, *bt.attend(return_lse=True))


@pytest.mark.parametrize("page", [1, 2, 5, 8, 16, 24, 48, 63, 64, 96, 100, 128, 1000])
def test_attend_pages(page):
    bt = Batch([1, page, page + 1, 64, 500, max(1, page - 1)], 16, page=page, dtype="fp16", seed=page)
    check_attend(bt, *bt.attend(return_lse=True))


@pytest.mark.parametrize("n", [1, 2, 63, 64, 65, 127, 128, 129, 191, 193, 4097, 30001])
def test_attend_one_sequence(n):
    bt = Batch([n], 33, page=16, seed=n)
    check_attend(bt, *bt.attend(return_lse=True))


@pytest.mark.parametrize("lens", [[0], [0, 0, 0], [1] * 300, [0] * 150 + [2000] + [0] * 150, [5000, 1, 0, 4000, 70],
                                  [(37 * i) % 400 for i in range(250)], [128] * 148, [64 * 149], [(11 * i) % 193 for i in range(300)]],
                         ids=["none", "all_empty", "many_single", "one_among_empty", "uneven", "250", "148", "149_tiles", "short"])
@pytest.mark.parametrize("heads,page", [(16, 16), (70, 5)])
def test_attend_batches(lens, heads, page):
    bt = Batch(lens, heads, dv=256, page=page, seed=len(lens))
    check_attend(bt, *bt.attend(return_lse=True))
    if max(lens) <= 192:  # no sequence can be split then, and a single kernel does all
        score = torch.rand(len(lens), bt.capacity, generator=bt.g, device="cuda")
        before = score.clone()
        out, lse = bt.attend(return_lse=True, score=score, max_len=max(max(lens), 1))
        check_attend(bt, out, lse, score, before)


def test_attend_thousands_of_sequences():
    lens = [37 * i % 130 for i in range(3000)]
    lens[1234] = 9000
    bt = Batch(lens, 4, 128, 0, 16, seed=1)
    check_attend(bt, *bt.attend(return_lse=True))


@pytest.mark.parametrize("heads,lens", [(16, [300, 0, 1, 64, 1000]), (128, [2049, 65, 3]), (70, [4000]), (3, [1] * 200)])
@pytest.mark.parametrize("dtype", TYPES)
def test_attend_score(heads, lens, dtype):
    bt = Batch(lens, heads, dtype=dtype, page=16, seed=heads)
    score0 = torch.rand(len(lens), bt.capacity + 5, generator=bt.g, device="cuda")[:, :bt.capacity + 2]
    score_out = torch.rand(len(lens), bt.capacity, generator=bt.g, device="cuda")
    want_out = score_out.clone()
    out, lse = bt.attend(return_lse=True, score=score0, score_out=score_out)
    for i, n in enumerate(lens):  # entries behind the last row stay as they were
        assert torch.equal(score_out[i, n:], want_out[i, n:])
        want_out[i, :n] = score0[i, :n]
    check_attend(bt, out, lse, score_out, want_out)
    # in place, the scratch sized for the longest sequence, and the same result without and with the weights
    again = score0.clone()
    assert torch.equal(bt.attend(score=again, max_len=max(lens)), out)
    for i, n in enumerate(lens):
        assert torch.equal(again[i, :n], score_out[i, :n]) and torch.equal(again[i, n:], score0[i, n:])
    assert torch.equal(bt.attend(), out)


def test_attend_strided_tensors():
    """A layer of a cache of several layers, slots before pages, a query and an output inside wider buffers."""
    lens = [200, 31, 0, 96]
    plain = Batch(lens, 24, dv=256, page=16, seed=3)
    want, want_lse = plain.attend(return_lse=True)
    pages, page, d = plain.cache.shape
    layers = torch.full((pages, 3, page, d + 8), NAN, dtype=torch.bfloat16, device="cuda")
    layered = Batch(lens, 24, dv=256, page=16, seed=3, cache=layers[:, 1, :, :d])
    got, lse = layered.attend(return_lse=True)
    assert torch.equal(got, want) and torch.equal(lse, want_lse)
    turned = Batch(lens, 24, dv=256, page=16, seed=3, cache=torch.empty(page, pages, d, dtype=torch.bfloat16, device="cuda").transpose(0, 1))
    wide = torch.full((24, 4, d + 264), 7.0, dtype=torch.bfloat16, device="cuda").transpose(0, 1)
    wide[..., :d] = turned.q
    turned.q = wide[..., :d]
    out = wide[..., d:d + 256]
    assert turned.attend(out=out) is out
    assert torch.equal(out, want) and (wide[..., d + 256:] == 7).all() and torch.equal(wide[..., :d], plain.q)
    odd = torch.full((4, 24, 259), 7.0, dtype=torch.bfloat16, device="cuda")
    plain.attend(out=odd[..., 1:257])
    assert torch.equal(odd[..., 1:257], want) and (odd[..., 257:] == 7).all() and (odd[..., :1] == 7).all()


def test_attend_lengths_and_pages_that_do_not_exist():
    # beyond the table: all its slots (the second sequence's table is full of its own pages, the rows behind are NaN)
    cut = Batch([96, 96], 16, dv=128, page=32, seed=6)
    cut.table = cut.table[:, :3].contiguous()
    want = cut.attend()
    cut.lens.fill_(10 ** 9)
    assert torch.equal(cut.attend(), want)
    # max_len cuts
    cut.lens.fill_(96)
    short = Batch([96, 96], 16, dv=128, page=32, seed=6)
    short.lens.fill_(50)
    assert torch.equal(cut.attend(max_len=50), short.attend())
    # negative: none
    bt = Batch([40, 80, 64, 100], 16, dv=128, page=32, seed=5)
    bt.lens[1] = -3
    bt.rows[1] = bt.rows[1][:0]
    check_attend(bt, *bt.attend(return_lse=True))
    # pages outside the cache read as zeros
    bt.table[3, 1], bt.table[2, 0] = -1, len(bt.cache)
    bt.rows[3][32:64], bt.rows[2][:32] = 0, 0
    check_attend(bt, *bt.attend(return_lse=True))


def test_attend_infinities_and_nan():
    bt = Batch([200, 200, 200], 16, dv=128, page=16, seed=8)
    out = bt.attend()
    ids = bt.table[:, :].long()
    bt.cache[ids[0, 9], 3] = NAN          # slot 147 of the first sequence
    bt.q[1, 4] = 0
    bt.q[1, 4, 0] = math.inf              # one head of the second: logits of +-inf
    got = bt.attend()
    assert torch.isnan(got[0]).all()
    assert torch.isnan(got[1, 4]).all()
    keep = [h for h in range(16) if h != 4]
    assert torch.equal(got[1, keep], out[1, keep]) and torch.equal(got[2], out[2])
    # a logit of -inf in the first tile gives that row no weight
    bt = Batch([130], 16, dv=128, dr=64, page=16, seed=9)
    bt.q[0, :, 128] = 1.0
    bt.rows[0][:70, 128] = -math.inf
    slot = torch.arange(70, device="cuda")
    bt.cache[bt.table[0].long()[slot // 16], slot % 16, 128] = -math.inf
    got = bt.attend()
    bt.rows[0] = bt.rows[0][70:]
    check_attend(bt, got)


@pytest.mark.parametrize("heads", [16, 64])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("first", [True, False])
def test_attend_a_long_tail(heads, dtype, first):
    """One row far above 20000 others whose weights, 2^-26 of it, are small numbers of fp16, and whose values outweigh its own. fp16
    weights are kept as multiples of 2^-24, with the largest at 2^7 or more: an error of 2^-32 of the largest weight for each row."""
    n = 20001
    bt = Batch([n], heads, page=64, dtype=dtype)
    bt.q.zero_()
    bt.q[:, :, bt.dv] = 1
    x = torch.zeros(n, bt.d, dtype=bt.dtype, device="cuda")
    hot = 0 if first else n - 1
    x[:, :bt.dv] = 1000
    x[:, bt.dv] = -250
    x[hot] = 2.0 ** -10
    slot = torch.arange(n, device="cuda")
    bt.cache[bt.table[0, slot // bt.page].long(), slot % bt.page] = x
    p = torch.softmax(bt.scale * x[:, bt.dv].double(), 0)
    want, u = p @ x[:, :bt.dv].double(), half_step(bt.dtype)
    ds = bt.scale * (bt.d + 2) * 2.0 ** -23 * 250
    tol = want * (2 * u + u * u + 2 * ds + 2.0 ** -20) + 2.0 ** -32 * n * 1000 * (bt.dtype == torch.float16)
    assert float(tol.max() / want.min()) < 0.02
    assert ((bt.attend()[0].double() - want).abs() <= tol).all()


@pytest.mark.parametrize("heads", [16, 40, 64])
@pytest.mark.parametrize("dtype", TYPES)
def test_attend_rising_and_falling_logits(heads, dtype):
    """Every tile far above the one before for some heads, far below for the others."""
    bt = Batch([1500, 30], heads, 256, 64, 48, dtype, seed=heads)
    bt.q[:, ::2, 256] = 2
    bt.q[:, 1::2, 256] = -2
    for i, x in enumerate(bt.rows):
        slot = torch.arange(len(x), device="cuda")
        x[:, 256] = (slot // 7 * 7).to(x.dtype)
        bt.cache[bt.table[i, slot // bt.page].long(), slot % bt.page] = x
    score = bt.slots(1.0)
    before = score.clone()
    out, lse = bt.attend(score=score, return_lse=True)
    check_attend(bt, out, lse, score, before)


@pytest.mark.parametrize("scale", [0.0, -0.05, 3.0])
def test_attend_scales(scale):
    """No preference, the least alike rows, nearly one row alone; the running maximum rises along the cache in the last."""
    bt = Batch([700, 64], 16, dv=128, page=64, seed=10)
    bt.scale = scale
    order = torch.argsort((bt.rows[0].double() @ bt.q[0, 0].double()) * (scale or 1))
    bt.rows[0] = bt.rows[0][order].contiguous()
    slot = torch.arange(700, device="cuda")
    bt.cache[bt.table[0].long()[slot // 64], slot % 64] = bt.rows[0]
    score = bt.slots()
    out, lse = bt.attend(return_lse=True, score=score)
    check_attend(bt, out, lse, score, bt.slots())


def test_attend_far_pages():
    """Rows past element 2^31 of the cache."""
    d, page = 576, 64
    pages = (1 << 31) // (page * d) + 40
    cache = torch.empty(pages, page, d, dtype=torch.bfloat16, device="cuda")
    bt = Batch([150, 10], 16, page=page, seed=11)
    want = bt.attend()
    small = bt.cache.clone()
    cache[-len(small):] = small
    bt.cache = cache
    bt.table = torch.where((bt.table >= 0) & (bt.table < len(small)), bt.table + (pages - len(small)), bt.table)
    assert torch.equal(bt.attend(), want)


def test_attend_repeats_to_the_bit():
    bt = Batch([9000, 3, 400, 0, 5000], 64, page=64, seed=12)
    score = bt.slots(1.0)
    first = bt.attend(return_lse=True, score=score)
    for _ in range(5):
        s = bt.slots(1.0)
        got = bt.attend(return_lse=True, score=s)
        assert torch.equal(got[0], first[0]) and torch.equal(got[1], first[1]) and torch.equal(s, score)


def test_streams_and_captured_graphs():
    """Two calls on two streams at once, two graphs captured on one stream and replayed on two: no scratch in common."""
    bts = [Batch([8000, 100, 0, 2000], 48, page=64, seed=20 + i) for i in range(2)]
    scores = [bt.slots() for bt in bts]
    want = [bt.attend(return_lse=True, score=s) for bt, s in zip(bts, scores)]
    streams = [torch.cuda.Stream() for _ in bts]
    torch.cuda.synchronize()
    got = [[] for _ in bts]
    for _ in range(10):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                s = torch.zeros_like(scores[i])
                o, l = pkg.mla_cache_attend(bts[i].q, bts[i].cache, bts[i].table, bts[i].lens, 512, bts[i].scale, score=s, return_lse=True)
                got[i].append((o, l, s))
    torch.cuda.synchronize()
    for i in range(2):
        for o, l, s in got[i]:
            assert torch.equal(o, want[i][0]) and torch.equal(l, want[i][1]) and torch.equal(s, scores[i])
    graphs, outs = [], []
    one = torch.cuda.Stream()
    for bt in bts:
        graph = torch.cuda.CUDAGraph()
        s = bt.slots()
        with torch.cuda.graph(graph, stream=one):
            s.zero_()
            o, l = pkg.mla_cache_attend(bt.q, bt.cache, bt.table, bt.lens, 512, bt.scale, score=s, return_lse=True)
        graphs.append(graph)
        outs.append((o, l, s))
    for _ in range(10):
        for graph, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                graph.replay()
    torch.cuda.synchronize()
    for i, (o, l, s) in enumerate(outs):
        assert torch.equal(o, want[i][0]) and torch.equal(l, want[i][1]) and torch.equal(s, scores[i])
    # new lengths in the same buffers are seen by the next replay
    bts[0].lens.copy_(torch.tensor([10, 0, 0, 64]))
    graphs[0].replay()
    torch.cuda.synchronize()
    bts[0].rows = [r[:n] for r, n in zip(bts[0].rows, (10, 0, 0, 64))]
    check_attend(bts[0], outs[0][0], outs[0][1])
    check_device_status()


# ---------------------------------------------------------------------------------------------------------------------


def turned(x, position, dv, theta):
    """x [..., d] in 64 bits with its last d - dv elements rotated, and the sum of the magnitudes that meet in each element."""
    half = (x.shape[-1] - dv) // 2
    y, mass = x.double().clone(), torch.zeros_like(x, dtype=torch.float64)
    if half:
        t = torch.arange(half, device=x.device, dtype=torch.float64)
        a = position * theta ** (-t / half)
        u, v = x[..., dv:dv + half].double(), x[..., dv + half:].double()
        y[..., dv:dv + half] = u * torch.cos(a) - v * torch.sin(a)
        y[..., dv + half:] = v * torch.cos(a) + u * torch.sin(a)
        mass[..., dv:dv + half] = mass[..., dv + half:] = u.abs() + v.abs()
    return y, mass


def assert_turned(got, x, position, dv, theta=10000.0):
    want, mass = turned(x, position, dv, theta)
    tol = half_step(x.dtype) * want.abs() + 2.0 ** -20 * mass + (mass > 0) * 1e-7 * (x.dtype == torch.float16)
    err = (got.double() - want).abs()
    assert (err <= tol).all(), float((err / tol.clamp_min(1e-30)).max())
    assert torch.equal(got[..., :dv], x[..., :dv])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dv,dr,heads,theta", [(512, 64, 16, 10000.0), (512, 64, 1, 1e6), (512, 64, 128, 10000.0), (384, 128, 5, 500.0),
                                               (128, 448, 7, 10000.0), (256, 0, 3, 10000.0)])
def test_append(dv, dr, heads, theta, dtype):
    lens = [0, 5, 16, 31, 47, 1]
    bt = Batch(lens, heads, dv, dr, 16, dtype, seed=heads, spare=16)
    b = len(lens)
    row = torch.randn(b, bt.d, generator=bt.g, device="cuda").to(bt.dtype)
    position = torch.tensor([0, 5, 4096, 199999, 1048575, 2 ** 31 - 1], dtype=torch.int32, device="cuda")
    score, at = bt.slots(3.0), bt.slots(9, torch.int32)
    before, q0 = bt.cache.clone(), bt.q.clone()
    q_out = torch.full_like(bt.q, NAN)
    assert pkg.mla_cache_append(row, position, bt.cache, bt.table, bt.lens, dv, theta, bt.q, q_out, score, at) is q_out
    assert torch.equal(bt.q, q0)
    for i, n in enumerate(lens):
        page, slot = int(bt.table[i, n // 16]), n % 16
        assert_turned(bt.cache[page, slot], row[i], int(position[i]), dv, theta)
        assert_turned(q_out[i], bt.q[i], int(position[i]), dv, theta)
        before[page, slot] = bt.cache[page, slot]
        assert score[i, n] == 0 and at[i, n] == position[i]
        score[i, n], at[i, n] = 3.0, 9
    assert torch.equal(bt.cache.view(torch.int16), before.view(torch.int16)) and (score == 3).all() and (at == 9).all()
    # in place, with nothing else asked for
    assert pkg.mla_cache_append(row, position, bt.cache, bt.table, bt.lens, dv, theta, bt.q) is bt.q
    assert torch.equal(bt.q, q_out) and torch.equal(bt.cache.view(torch.int16), before.view(torch.int16))
    assert pkg.mla_cache_append(row, position, bt.cache, bt.table, bt.lens, dv, theta) is None


def test_append_rows_off_16_bytes_and_sequences_left_alone():
    lens = [3, 20, 40, 7, 30]
    bt = Batch(lens, 6, 128, 64, 16, seed=2, spare=16)
    wide = torch.randn(5, 9, bt.d + 3, generator=bt.g, device="cuda").to(bt.dtype)
    row, q = wide[:, 0, 1:bt.d + 1], wide[:, 1:7, 2:bt.d + 2]
    position = torch.arange(5, dtype=torch.int32, device="cuda") * 1000
    q_out = torch.zeros(5, 6, bt.d + 1, dtype=bt.dtype, device="cuda")[..., :bt.d]
    bt.lens.copy_(torch.tensor([3, -1, 10 ** 9, 7, bt.capacity]))
    bt.table[3, 0] = len(bt.cache)
    before = bt.cache.clone()
    score = bt.slots(3.0)
    pkg.mla_cache_append(row, position, bt.cache, bt.table, bt.lens, 128, q=q, q_out=q_out, score=score)
    page = int(bt.table[0, 0])
    assert_turned(bt.cache[page, 3], row[0], 0, 128)
    for i in range(5):
        assert_turned(q_out[i], q[i], 1000 * i, 128)
    before[page, 3] = bt.cache[page, 3]
    assert torch.equal(bt.cache.view(torch.int16), before.view(torch.int16))
    assert score[0, 3] == 0 and int((score != 3).sum()) == 1


# ---------------------------------------------------------------------------------------------------------------------


def evicted(score, position, n, budget, recent):
    """Slot of the row that each slot below the new length holds afterwards."""
    if n <= budget:
        return list(range(n))
    score, position = score[:n].tolist(), position[:n].tolist()
    newest = max(position)
    safe = [p > newest - recent for p in position]

    order = sorted(range(n), key=lambda j: (0, 0, 0.0, j) if safe[j] else (1, 0, 0.0, j) if score[j] != score[j] else (1, 1, -score[j], j))
    stays = set(order[:budget])
    late = iter(sorted(j for j in stays if j >= budget))
    return [j if j in stays else next(late) for j in range(budget)]


def run_evict(lens, budget, recent, page=16, dv=128, dtype="bf16", seed=0, make=None, in_place=False):
    bt = Batch(lens, 1, dv, 64, page, dtype, seed=seed)
    score = (2 * torch.randn(len(lens), bt.capacity, generator=bt.g, device="cuda")).exp()
    position = torch.arange(bt.capacity, dtype=torch.int32, device="cuda").repeat(len(lens), 1)
    if make:
        make(score, position)
    s0, p0, c0, l0 = score.clone(), position.clone(), bt.cache.clone(), bt.lens.clone()
    outs = {} if in_place else dict(lens_out=torch.full_like(bt.lens, -1), score_out=torch.full_like(score, 5.0),
                                    position_out=torch.full_like(position, 6))
    got = pkg.mla_cache_evict(bt.cache, bt.table, bt.lens, score, position, budget, recent, **outs)
    assert got is outs.get("lens_out", bt.lens)
    so, po = outs.get("score_out", score), outs.get("position_out", position)
    assert got.tolist() == [min(n, budget) for n in lens]
    want_s, want_p, want_c = (s0.clone(), p0.clone(), c0.clone()) if in_place else (torch.full_like(score, 5.0), torch.full_like(position, 6), c0.clone())
    table = bt.table.cpu()
    for i, n in enumerate(lens):
        took = evicted(s0[i], p0[i], n, budget, recent)
        assert len(took) == min(n, budget)
        at = torch.tensor(took, dtype=torch.long, device="cuda")
        want_s[i, :len(took)], want_p[i, :len(took)] = s0[i, at], p0[i, at]
        for j, src in enumerate(took):
            if j != src:
                want_c[int(table[i, j // page]), j % page] = c0[int(table[i, src // page]), src % page]
    assert torch.equal(so.view(torch.int32), want_s.view(torch.int32)) and torch.equal(po, want_p)
    assert torch.equal(bt.cache.view(torch.int16), want_c.view(torch.int16))
    if not in_place:
        assert torch.equal(bt.lens, l0) and torch.equal(score.view(torch.int32), s0.view(torch.int32)) and torch.equal(position, p0)
    return bt, score, position, outs


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("lens,budget,recent", [([65, 64, 10, 0, 1], 64, 16), ([200, 1000, 33], 32, 32), ([200, 1000, 33], 32, 0),
                                                ([2, 1], 1, 1), ([2, 1], 1, 0), ([3000], 2999, 100), ([5000, 5000], 700, 50),
                                                ([17] * 40, 5, 2), ([100], 1 << 30, 5)])
def test_evict(lens, budget, recent, in_place):
    run_evict(lens, budget, recent, in_place=in_place)


@pytest.mark.parametrize("page,dv,dtype", [(1, 128, "bf16"), (7, 256, "fp16"), (24, 512, "bf16"), (64, 384, "fp16")])
def test_evict_pages_and_rows(page, dv, dtype):
    run_evict([333, 90, 20], 40, 10, page, dv, dtype, seed=page)


def test_evict_ties_zeros_nan_infinities():
    def equal(score, position):
        score.fill_(0.25)

    def mixed(score, position):
        score[:, ::3] = 0.0
        score[:, 1::3] = -0.0
        score[0, 5:200:7] = NAN
        score[1, 5:200:7] = math.inf
        score[2, 5:200:7] = -math.inf
        score[2, 6:200:7] = -1.5

    def shuffled(score, position):
        g = torch.Generator(device="cuda").manual_seed(4)
        position.copy_(torch.argsort(torch.rand(score.shape, generator=g, device="cuda"), dim=1).int() * 5)

    for make in (equal, mixed, shuffled):
        for budget, recent in ((50, 10), (30, 0), (60, 60)):
            run_evict([200, 201, 300], budget, recent, make=make)

    def ends(score, position):  # positions at both ends of the type
        position[:, :100] = -2 ** 31
        position[:, 150] = 2 ** 31 - 1
    run_evict([200, 201, 300], 50, 50, make=ends)


@pytest.mark.parametrize("n", [1023, 1025, 40000, 131072])
def test_evict_long(n):
    run_evict([n, n // 2], 1000, 100, page=64, seed=n)


@pytest.mark.parametrize("lens,budget", [([700, 650, 90], 300), ([9000, 8000], 4100), ([40000], 1500)])
@pytest.mark.parametrize("spread", ["equal", "two", "neighbours", "outliers", "dense", "one position", "denormal"])
def test_evict_spreads_of_the_scores(spread, lens, budget):
    """Ranges of the scores from one value to all there are, with many rows at the border or none."""
    def make(score, position):
        g = torch.Generator(device="cuda").manual_seed(len(lens))
        k = torch.randint(0, 5000, score.shape, generator=g, device="cuda")
        near = torch.full_like(score, 1.0).view(torch.int32)
        if spread == "equal":
            score.fill_(-3.0)
        elif spread == "two":
            score.copy_((k % 2).float())
        elif spread == "neighbours":
            score.copy_((near + (k % 300).int()).view(torch.float32))
        elif spread == "outliers":
            score.copy_((near + k.int()).view(torch.float32))
            for n, v in ((0, math.inf), (1, -math.inf), (2, NAN), (3, -1e38), (4, 0.0)):
                score[:, n::613] = v
        elif spread == "dense":  # a bin that holds most of the rows
            score.copy_(torch.where(k < 4000, (near + k.int()).view(torch.float32), score))
        elif spread == "one position":  # all rows are protected, more than stay
            position.fill_(-7)
        else:
            score.copy_((k.int() - 2500).abs().view(torch.float32) * (1 - 2 * (k % 2)))
    run_evict(lens, budget, budget // 4, page=64, seed=budget, make=make, in_place=True)


def test_evict_a_second_time_changes_nothing():
    bt, score, position, outs = run_evict([500, 60], 100, 10)
    before = bt.cache.clone()
    pkg.mla_cache_evict(bt.cache, bt.table, outs["lens_out"], outs["score_out"], outs["position_out"], 100, 10)
    assert torch.equal(bt.cache.view(torch.int16), before.view(torch.int16)) and outs["lens_out"].tolist() == [100, 60]


# ---------------------------------------------------------------------------------------------------------------------


def test_empty_batch():
    bt = Batch([5], 4, 128, 64, 16)
    none = slice(0, 0)
    out, lse = pkg.mla_cache_attend(bt.q[none], bt.cache, bt.table[none], bt.lens[none], 128, 0.1, return_lse=True)
    assert out.shape == (0, 4, 128) and lse.shape == (0, 4)
    pkg.mla_cache_append(bt.q[none, 0], bt.lens[none], bt.cache, bt.table[none], bt.lens[none], 128)
    pkg.mla_cache_evict(bt.cache, bt.table[none], bt.lens[none], bt.slots()[none], bt.slots(0, torch.int32)[none], 3, 1)


@pytest.mark.parametrize("captured", [False, True])
def test_decode_loop(captured):
    """The operators as a decode loop runs them, steps on end: projection, append, attend with weights, evict. After each step
    the attention is checked against the rows that the cache should hold, and the eviction against the scores it was given."""
    heads, dv, dr, page, budget, recent, k = 16, 512, 64, 16, 96, 20, 512
    lens0 = [94, 96, 40, 95, 0]
    b = len(lens0)
    bt = Batch(lens0, heads, dv, dr, page, seed=31, spare=40)
    score, at = bt.slots(), bt.slots(0, torch.int32)
    at[:] = torch.arange(bt.capacity, device="cuda")
    position = bt.lens.clone()
    rows = [list(r) for r in bt.rows]
    w, ws = pkg.make_inputs(b, dv + dr, k, seed=5, device="cuda")[1], pkg.make_inputs(b, dv + dr, k, seed=5, device="cuda")[3]
    x, xs = pkg.make_inputs(b, dv + dr, k, seed=6, device="cuda")[0], pkg.make_inputs(b, dv + dr, k, seed=6, device="cuda")[2]
    row, q = torch.empty(b, dv + dr, dtype=torch.bfloat16, device="cuda"), bt.q.clone()
    q_out, out = torch.empty_like(q), torch.empty(b, heads, dv, dtype=torch.bfloat16, device="cuda")
    seen = torch.empty_like(score)

    def step():
        pkg.kv_down_projection_fp8(x, xs, w, ws, out=row)
        pkg.mla_cache_append(row, position, bt.cache, bt.table, bt.lens, dv, q=q, q_out=q_out, score=score, slot_position=at)
        bt.lens.add_(1)
        position.add_(1)
        pkg.mla_cache_attend(q_out, bt.cache, bt.table, bt.lens, dv, bt.scale, out=out, score=score)
        seen.copy_(score)
        pkg.mla_cache_evict(bt.cache, bt.table, bt.lens, score, at, budget, recent)

    state = [bt.cache, bt.lens, score, at, position]
    saved = [t.clone() for t in state]
    if captured:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        for t, s in zip(state, saved):
            t.copy_(s)
    for n_step in range(4):
        at0, pos0 = at.clone(), position.clone()
        x.copy_(pkg.make_inputs(b, dv + dr, k, seed=40 + n_step, device="cuda")[0])
        graph.replay() if captured else step()
        for i in range(b):
            # The new row as the cache holds it: slots behind the budget keep what they had. Its rotation may round the other
            # way than the 64-bit one.
            n = len(rows[i])
            held = bt.cache[bt.table[i].long()[n // page], n % page]
            assert_turned(held, row[i], int(pos0[i]), dv)
            assert_turned(q_out[i], q[i], int(pos0[i]), dv)
            rows[i].append(held.clone())
            at0[i, n] = pos0[i]
            one = Batch.__new__(Batch)
            one.__dict__.update(bt.__dict__)
            one.q, one.rows = q_out[i:i + 1], [torch.stack(rows[i])]
            check_attend(one, out[i:i + 1])
        for i in range(b):
            n = len(rows[i])
            took = evicted(seen[i], at0[i], n, budget, recent)
            rows[i] = [rows[i][j] for j in took]
            assert int(bt.lens[i]) == len(took)
            slot = torch.arange(len(took), device="cuda")
            held = bt.cache[bt.table[i].long()[slot // page], slot % page]
            assert torch.equal(held, torch.stack(rows[i]))
            assert torch.equal(at[i, :len(took)], at0[i, torch.tensor(took, device="cuda")])
    check_device_status()


def test_results_without_the_native_module(monkeypatch):
    """The Python checks and ctypes calls do what the native module does."""
    from amd_developer_challenge_2025_b200 import _lib

    def all_calls():
        bt = Batch([70, 0, 33], 5, 128, 64, 16, seed=41, spare=16)
        score, at = bt.slots(1.0), bt.slots(0, torch.int32)
        at[:] = torch.arange(bt.capacity, device="cuda")
        row = torch.randn(3, bt.d, generator=bt.g, device="cuda").to(bt.dtype)
        found = [pkg.mla_cache_append(row, bt.lens.clone(), bt.cache, bt.table, bt.lens, 128, 5000.0, bt.q, torch.empty_like(bt.q), score, at)]
        bt.lens += 1
        found += [*bt.attend(return_lse=True, score=score, max_len=80), bt.attend(out=torch.empty(3, 5, 128, dtype=bt.dtype, device="cuda"))]
        found += [pkg.mla_cache_evict(bt.cache, bt.table, bt.lens, score, at, 20, 4), score, at, bt.cache.nan_to_num(7.0)]
        return found

    want = all_calls()
    monkeypatch.setattr(_lib, "_host", _lib._PythonChecks)
    for g, w in zip(all_calls(), want):
        assert g.shape == w.shape and g.dtype == w.dtype and torch.equal(g, w)


@pytest.mark.parametrize("batch,n,budget", [(1, 70001, 30000), (3, 9000, 4000), (20, 5000, 64), (150, 300, 290), (1, 300000, 17), (75, 21000, 20930)])
def test_evict_shapes_of_clusters(batch, n, budget):
    run_evict([n - i for i in range(batch)], budget, budget // 3, page=64, seed=n, in_place=True)


@pytest.mark.parametrize("lens", [[130, 0, 64], [4000, 100, 0, 60]], ids=["whole", "split"])
@pytest.mark.parametrize("heads,page,dtype", [(16, 16, "bf16"), (16, 5, "fp16"), (40, 16, "fp16"), (128, 64, "bf16")])
def test_attend_heads_without_weights(lens, heads, page, dtype):
    """A head all of whose logits are -inf gets zeros and an lse of -inf, as a sequence without rows does, and adds nothing to the
    scores; the other heads of its sequence are as they would be without it."""
    bt = Batch(lens, heads, dv=128, page=page, dtype=dtype, seed=heads)
    for i, x in enumerate(bt.rows):
        slot = torch.arange(len(x), device="cuda")
        x[:, 130] = 1.0
        bt.cache[bt.table[i, slot // page].long(), slot % page] = x
    dead = torch.arange(heads, device="cuda") % 5 == 2
    bt.q[:, dead, 130] = -math.inf
    score = torch.rand(len(lens), bt.capacity, generator=bt.g, device="cuda")
    before = score.clone()
    out, lse = bt.attend(return_lse=True, score=score, max_len=max(lens))
    assert (out[:, dead] == 0).all() and (lse[:, dead] == -math.inf).all()
    live = Batch.__new__(Batch)
    live.__dict__.update(bt.__dict__)
    live.q = bt.q[:, ~dead]
    check_attend(live, out[:, ~dead], lse[:, ~dead], score, before)
    # every head of every sequence: the scores stay as they were
    bt.q[:, :, 130] = -math.inf
    score.copy_(before)
    out, lse = bt.attend(return_lse=True, score=score)
    assert (out == 0).all() and (lse == -math.inf).all() and torch.equal(score, before)


@pytest.mark.parametrize("heads", [64 * 148 + 1, 1 << 16])
def test_attend_more_head_tiles_than_sms(heads):
    """Every head tile has one worker then, and the launch more CTAs than the chip takes at a time."""
    bt = Batch([400, 0, 33], heads, dv=128, dr=0, page=16, seed=3)
    score = bt.slots()
    out, lse = bt.attend(return_lse=True, score=score, max_len=400)
    check_attend(bt, out, lse, score, bt.slots())


@pytest.mark.parametrize("heads", [16, 40, 128])
@pytest.mark.parametrize("page", [16, 5])
def test_attend_an_expired_wait_is_reported_and_the_context_stays_usable(heads, page):
    """In the allowed form: every wait is limited to 5 ms, a tile is not copied, the kernel gives up by itself and says which wait it was.
    The next ordinary call, which finds shared memory and TMEM as that one left them, is right."""
    from amd_developer_challenge_2025_b200.mla_cache import selftest_wait_expiry

    check_device_status()
    words = selftest_wait_expiry("cuda", heads, page)
    assert words[0] == 1 and 0x201 <= words[1] <= 0x205, [hex(w) for w in words]
    bt = Batch([300, 0, 1, 2000], heads, page=page, seed=heads)
    check_attend(bt, *bt.attend(return_lse=True))
