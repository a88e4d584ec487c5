"""Cases of the operators around a paged latent cache: append, attend, evict.

    own                 False: `run` computes the plain form in torch; True: it calls the package
    listed()            the standing cases
    draw(rng)           one more case of the same ranges
    prepare(case, seed) what a decode loop has in hand before the call
    run(state)          one call and its outputs
    work(case)          bytes and operations one call cannot do without
    exact(case, seed)   the outputs of that call in 64 bits

The cache is [pages, page_size, dv + dr]: slot j of sequence b lies in page block_table[b, j // page_size]. A row is the key of
every query head, its first dv elements are the value. Kinds of case ("op"):

* append   the new row of every sequence goes to the slot behind its last one, its last dr elements rotated for the sequence's
           own position, as are those of the query heads
* attend   one new token of every sequence attends to its cached rows; with "score", the weights that every slot received are
           added up over the heads
* evict    sequences longer than a budget keep the rows of the newest positions and those of the largest accumulated weight
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
THETA = 10000.0
NOPE = 128  # width of a query head before the up-projection is folded into it: the softmax scale is that of NOPE + dr
MAX_ROWS = 128 * 4096  # cached rows of the largest case
MAX_SCORE_ROWS = 32 * 4096  # and of the largest one that adds up weights


def append(name, b, nh, dtype="bf16", dv=512, dr=64, page=16, rows=64):
    return {"name": name, "op": "append", "b": b, "nh": nh, "dtype": dtype, "dv": dv, "dr": dr, "page": page, "rows": rows}


def attend(name, b, nh, rows, spread="equal", dtype="bf16", dv=512, dr=64, page=64, score=False):
    return {"name": name, "op": "attend", "b": b, "nh": nh, "rows": rows, "spread": spread, "dtype": dtype, "dv": dv, "dr": dr,
            "page": page, "score": score}


def evict(name, b, rows, budget, recent, spread="equal", dtype="bf16", dv=512, dr=64, page=64):
    return {"name": name, "op": "evict", "b": b, "rows": rows, "budget": budget, "recent": recent, "spread": spread,
            "dtype": dtype, "dv": dv, "dr": dr, "page": page}


def listed():
    return [
        # One sequence, few heads (a shard of a model over several GPUs): call and launch overhead are most of it.
        append("append_b1_h16", 1, 16),
        # A full decode batch with all heads: the query is most of the bytes.
        append("append_b128_h128", 128, 128),
        # A short chat turn of a single user: latency alone.
        attend("attend_b1_h16_77", 1, 16, 77, page=16),
        # One long document, all heads: the cache's length is all there is to split.
        attend("attend_b1_h128_65536", 1, 128, 65536),
        # A decode batch of a server: sequences of every length up to 8192, empty ones of a padded batch among them.
        attend("attend_b64_h128_ragged", 64, 128, 8192, "ragged"),
        # A wide batch on a shard with 16 of the heads, fp16: the cache's bytes are all that counts.
        attend("attend_b128_h16_4096", 128, 16, 4096, dtype="fp16", page=32),
        # Odd everything: heads that fill no tile, pages that end inside one, a narrower latent.
        attend("attend_b7_h40_odd", 7, 40, 3001, "ragged", dv=256, page=24),
        # A loop that evicts, few heads: the weights of one step.
        attend("attend_score_b8_h16", 8, 16, 2049, page=16, score=True),
        # The same with all heads over a ragged batch.
        attend("attend_score_b32_h128", 32, 128, 4096, "ragged", score=True),
        # Every step of that loop: one row too many in each sequence.
        evict("evict_step_b64", 64, 2049, 2048, 256, page=32),
        # Behind the prompts of a batch: most rows leave.
        evict("evict_prompt_b8", 8, 16384, 2048, 512, "ragged"),
        # One long document down to a sixteenth.
        evict("evict_long_b1", 1, 131072, 8192, 1024),
    ]


def _spread(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng: random.Random):
    op = rng.choice(["append", "attend", "attend", "attend", "evict"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    dv, dr = rng.choice([(512, 64), (512, 64), (256, 64), (128, 128)])
    page = rng.choice([8, 16, 24, 32, 40, 64, 64, 100, 128])
    spread = rng.choice(["equal", "ragged"])
    if op == "append":
        return append("", _spread(rng, 1, 128), _spread(rng, 1, 128), dtype, dv, dr, page, rng.randint(1, 64))
    if op == "attend":
        score = rng.random() < 0.4
        b = _spread(rng, 1, 128)
        most = (MAX_SCORE_ROWS if score else MAX_ROWS) // b
        return attend("", b, _spread(rng, 1, 128), _spread(rng, 1, min(most, 65536)), spread, dtype, dv, dr, page, score)
    b = _spread(rng, 1, 64)
    rows = _spread(rng, 64, min(131072, 131072 // b))
    budget = rng.choice([rows - 1, _spread(rng, 32, rows), _spread(rng, 32, rows)])
    return evict("", b, rows, budget, rng.randint(0, budget // 2), spread, dtype, dv, dr, page)


def lens_of(case):
    """Rows each sequence has. A ragged batch of three or more has an empty sequence and one of a single row."""
    b, rows = case["b"], case["rows"]
    if case["op"] == "append":
        return [(17 * i) % rows for i in range(b)]
    if case["spread"] == "equal":
        return [rows] * b
    rng = random.Random(1000003 * b + rows)
    lens = [rows] + [rng.randint(1, rows) for _ in range(b - 1)]
    if b >= 3:
        lens[1], lens[2] = 0, 1
    return lens


def capacity_of(case):
    """Slots the block table has room for: the longest sequence and a page more."""
    return (case["rows"] // case["page"] + 1) * case["page"]


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dtype = TYPES[case["dtype"]]
    b, ps, d = case["b"], case["page"], case["dv"] + case["dr"]
    per_seq = capacity_of(case) // ps
    lens = lens_of(case)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32)

    # Pages are handed out as sequences grow: a sequence's lie anywhere. Two pages of the pool are nobody's.
    pages = b * per_seq + 2
    st = {
        "case": case,
        "lens": torch.tensor(lens, dtype=torch.int32, device=DEV),
        "block_table": torch.randperm(pages, generator=g, device=DEV)[: b * per_seq].to(torch.int32).view(b, per_seq),
        "cache": torch.randn(pages, ps, d, generator=g, device=DEV, dtype=dtype),
    }
    if case["op"] == "append":
        st["row"] = normal(b, d).to(dtype)
        st["position"] = torch.randint(0, 200000, (b,), generator=g, device=DEV, dtype=torch.int32)
        st["q"] = normal(b, case["nh"], d).to(dtype)
        st["q_out"] = torch.zeros_like(st["q"])
        st["score"] = normal(b, per_seq * ps).abs()
        st["slot_position"] = torch.zeros(b, per_seq * ps, dtype=torch.int32, device=DEV)
    elif case["op"] == "attend":
        st["q"] = normal(b, case["nh"], d).to(dtype)
        st["scale"] = 1.0 / math.sqrt(NOPE + case["dr"])
        if case["score"]:
            st["score"] = normal(b, per_seq * ps).exp()
            st["score_out"] = torch.zeros_like(st["score"])
    else:
        # Accumulated weights spread over orders of magnitude; rows that came last have received none yet, so there are ties.
        score = (2 * normal(b, per_seq * ps)).exp()
        score[torch.rand(b, per_seq * ps, generator=g, device=DEV) < 0.02] = 0.0
        st["score"] = score
        pos = torch.arange(per_seq * ps, device=DEV, dtype=torch.int32).repeat(b, 1)
        if case["rows"] == case["budget"] + 1:
            # A loop that has evicted before: holes were filled, so slots are in no order but for the row that has just come.
            order = torch.argsort(torch.rand(b, case["budget"], generator=g, device=DEV), dim=1)
            pos[:, : case["budget"]] = 3 * order.to(torch.int32)
            pos[:, case["budget"]:] += 3 * case["budget"]
        st["slot_position"] = pos
        st["lens_out"] = torch.zeros_like(st["lens"])
        st["score_out"] = torch.zeros_like(score)
        st["position_out"] = torch.zeros_like(pos)
    return st


# ---------------------------------------------------------------------------------------------------------------------
# Plain forms
# ---------------------------------------------------------------------------------------------------------------------


def _rotated(x, position, dv):
    """x [B, ..., d] with its last d - dv elements rotated for position [B], in 32 bits; angles in 64."""
    half = (x.shape[-1] - dv) // 2
    freq = THETA ** (torch.arange(half, device=x.device, dtype=torch.float64) / -half)
    angle = position.double()[:, None] * freq
    angle = angle.view(angle.shape[0], *([1] * (x.dim() - 2)), half)
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    nope, x1, x2 = x[..., :dv].float(), x[..., dv:dv + half].float(), x[..., dv + half:].float()
    return torch.cat([nope, x1 * cos - x2 * sin, x2 * cos + x1 * sin], dim=-1)


def _append(st):
    case, cache, lens = st["case"], st["cache"], st["lens"].long()
    seqs = torch.arange(case["b"], device=cache.device)
    page = st["block_table"].long()[seqs, lens // case["page"]]
    cache[page, lens % case["page"]] = _rotated(st["row"], st["position"], case["dv"]).to(cache.dtype)
    st["q_out"].copy_(_rotated(st["q"], st["position"], case["dv"]))
    st["score"][seqs, lens] = 0.0
    st["slot_position"][seqs, lens] = st["position"]


def _rows(st, width):
    """The cached rows of every sequence, [B, width, d] in 32 bits, zero behind the last, and which of them exist."""
    case = st["case"]
    slot = torch.arange(width, device=st["cache"].device)
    exists = slot < st["lens"][:, None]
    page = st["block_table"].long()[:, slot // case["page"]]
    rows = st["cache"][page, slot % case["page"]].float()
    return rows.masked_fill_(~exists[..., None], 0.0), exists


def _attend(st):
    case = st["case"]
    rows, exists = _rows(st, case["rows"])
    s = torch.matmul(st["q"].float() * st["scale"], rows.transpose(1, 2)).masked_fill_(~exists[:, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = torch.exp(s - top)
    total = p.sum(-1, keepdim=True)
    lse = (top + torch.log(total)).squeeze(-1)
    p = p / torch.where(total == 0, torch.ones_like(total), total)
    out = torch.matmul(p, rows[..., : case["dv"]]).to(st["q"].dtype)
    if case["score"]:
        width = case["rows"]
        kept = st["score_out"][:, :width]
        kept.copy_(torch.where(exists, st["score"][:, :width] + p.sum(1), kept))
    return out, lse


def _evict(st):
    case, cache = st["case"], st["cache"]
    budget, ps = case["budget"], case["page"]
    lens = st["lens"].long()[:, None]
    width = case["rows"]
    score, position = st["score"][:, :width], st["slot_position"][:, :width]
    slot = torch.arange(width, device=cache.device)
    exists = slot < lens
    newest = torch.where(exists, position, torch.full_like(position, -1)).amax(1, keepdim=True)
    safe = exists & (position > newest - case["recent"])
    key = torch.where(safe, math.inf, torch.where(exists, score, -math.inf))
    order = torch.argsort(key, dim=1, descending=True, stable=True)
    kept = torch.zeros_like(exists).scatter_(1, order[:, :budget], True)
    kept = torch.where(lens > budget, kept, exists)
    first = exists & (slot < budget)
    lens_out = torch.clamp(lens, max=budget)
    src_slot = slot.repeat(case["b"], 1)
    to = (first & ~kept).nonzero(as_tuple=True)
    of = (kept & (slot >= budget) & (lens > budget)).nonzero(as_tuple=True)  # as many in each sequence, in the same order
    src_slot[to] = of[1]
    table = st["block_table"].long()
    cache[table[to[0], to[1] // ps], to[1] % ps] = cache[table[of[0], of[1] // ps], of[1] % ps]
    there = slot < lens_out
    st["lens_out"].copy_(lens_out[:, 0])
    score_out, position_out = st["score_out"][:, :width], st["position_out"][:, :width]
    score_out.copy_(torch.where(there, score.gather(1, src_slot), score_out))
    position_out.copy_(torch.where(there, position.gather(1, src_slot), position_out))


def run(state):
    st, case = state, state["case"]
    if case["op"] == "append":
        if own:
            import amd_developer_challenge_2025_b200 as pkg

            pkg.mla_cache_append(st["row"], st["position"], st["cache"], st["block_table"], st["lens"], case["dv"],
                                 theta=THETA, q=st["q"], q_out=st["q_out"], score=st["score"],
                                 slot_position=st["slot_position"])
        else:
            _append(st)
        return {k: st[k] for k in ("q_out", "cache", "score", "slot_position")}
    if case["op"] == "attend":
        if own:
            import amd_developer_challenge_2025_b200 as pkg

            out, lse = pkg.mla_cache_attend(st["q"], st["cache"], st["block_table"], st["lens"], case["dv"], st["scale"],
                                            score=st.get("score"), score_out=st.get("score_out"), max_len=case["rows"],
                                            return_lse=True)
        else:
            out, lse = _attend(st)
        found = {"out": out, "lse": lse}
        if case["score"]:
            found["score"] = st["score_out"]
        return found
    if own:
        import amd_developer_challenge_2025_b200 as pkg

        pkg.mla_cache_evict(st["cache"], st["block_table"], st["lens"], st["score"], st["slot_position"], case["budget"],
                            case["recent"], lens_out=st["lens_out"], score_out=st["score_out"],
                            position_out=st["position_out"])
    else:
        _evict(st)
    return {k: st[k] for k in ("cache", "lens_out", "score_out", "position_out")}


def work(case):
    b, d, lens = case["b"], case["dv"] + case["dr"], lens_of(case)
    rows = sum(lens)
    if case["op"] == "append":
        heads = b * case["nh"]
        return {"bytes": 2 * 2 * (b + heads) * d + b * (3 * 4 + 2 * 4), "flops": 3 * (b + heads) * case["dr"]}
    if case["op"] == "attend":
        heads = b * case["nh"]
        tables = 4 * (b + sum(-(-n // case["page"]) for n in lens))
        moved = 2 * rows * d + 2 * heads * (d + case["dv"]) + 4 * heads + tables
        return {"bytes": moved + (8 * rows if case["score"] else 0), "flops": 2 * case["nh"] * (d + case["dv"]) * rows}
    moves, written = 0.0, 0
    for n in lens:
        over = n - case["budget"]
        written += min(n, case["budget"])
        if over > 0:
            # Kept rows behind the budget: the newest, and of the others there the share that stays.
            newest = min(case["recent"], over) if case["recent"] else 0
            moves += newest + (over - newest) * (case["budget"] - case["recent"]) / max(1, n - case["recent"])
    return {"bytes": 8 * rows + 8 * written + round(2 * 2 * d * moves) + 8 * b, "flops": 8 * rows}


# ---------------------------------------------------------------------------------------------------------------------
# 64 bits, sequence by sequence from the definitions
# ---------------------------------------------------------------------------------------------------------------------


def exact(case, seed):
    def turned(x, position):
        half = (x.shape[-1] - dv) // 2
        y = x.double().clone()
        for t in range(half):
            a = position * THETA ** (-t / half)
            u, v = x[..., dv + t].double(), x[..., dv + half + t].double()
            y[..., dv + t] = u * math.cos(a) - v * math.sin(a)
            y[..., dv + half + t] = v * math.cos(a) + u * math.sin(a)
        return y

    st = prepare(case, seed)
    lens, ps, dv = lens_of(case), case["page"], case["dv"]
    table = st["block_table"].long()
    if case["op"] == "append":
        cpu = {k: st[k].cpu() for k in ("row", "q", "position", "block_table")}
        cache, q_out = st["cache"].double(), []
        for i, n in enumerate(lens):
            at = int(cpu["position"][i])
            cache[int(cpu["block_table"][i, n // ps]), n % ps] = turned(cpu["row"][i], at).to(DEV)
            q_out.append(turned(cpu["q"][i], at))
            st["score"][i, n] = 0.0
            st["slot_position"][i, n] = at
        return {"q_out": torch.stack(q_out).to(DEV), "cache": cache, "score": st["score"].double(),
                "slot_position": st["slot_position"]}
    flat = st["cache"].view(-1, st["cache"].shape[-1])
    if case["op"] == "attend":
        b, nh = case["b"], case["nh"]
        out = torch.zeros(b, nh, dv, dtype=torch.float64, device=DEV)
        lse = torch.full((b, nh), -math.inf, dtype=torch.float64, device=DEV)
        score = st["score_out"].double() if case["score"] else None
        for i, n in enumerate(lens):
            if n == 0:
                continue
            at = (table[i][:, None] * ps + torch.arange(ps, device=DEV)).view(-1)[:n]
            x = flat[at].double()
            s = (x @ st["q"][i].double().T) * st["scale"]  # [n, nh]
            lse[i] = torch.logsumexp(s, dim=0)
            w = torch.exp(s - lse[i])
            out[i] = w.T @ x[:, :dv]
            if case["score"]:
                score[i, :n] = st["score"][i, :n].double() + w.sum(1)
        found = {"out": out, "lse": lse}
        if case["score"]:
            found["score"] = score
        return found
    lens_out, score_out, position_out = list(lens), st["score_out"].double(), st["position_out"]
    for i, n in enumerate(lens):
        k = case["budget"]
        score, position = st["score"][i, :n].tolist(), st["slot_position"][i, :n].tolist()
        took = list(range(min(n, k)))
        if n > k:
            lens_out[i] = k
            newest = max(position)
            safe = [at > newest - case["recent"] for at in position]
            rank = sorted(range(n), key=lambda j: (not safe[j], 0.0 if safe[j] else -score[j], j))
            stays = set(rank[:k])
            late = iter(sorted(j for j in stays if j >= k))
            took = [j if j in stays else next(late) for j in range(k)]
            at = (table[i][:, None] * ps + torch.arange(ps, device=DEV)).view(-1)
            pairs = [(j, t) for j, t in enumerate(took) if j != t]
            if pairs:
                to, of = (torch.tensor(v, device=DEV) for v in zip(*pairs))
                flat[at[to]] = flat[at[of]]
        if took:
            score_out[i, : len(took)] = torch.tensor([score[j] for j in took], dtype=torch.float64, device=DEV)
            position_out[i, : len(took)] = torch.tensor([position[j] for j in took], dtype=torch.int32, device=DEV)
    return {"cache": st["cache"].double(), "lens_out": torch.tensor(lens_out, dtype=torch.int32, device=DEV),
            "score_out": score_out, "position_out": position_out}
