"""Operators around a paged latent cache, the part of an MLA decode step between the KV down-projection and the output
projection: a new row written into its page, the attention of one new token per sequence, and eviction by accumulated
attention weight.

The cache is a tensor [pages, page_size, dv + dr] (bf16 or fp16): slot j of sequence b is row
cache[block_table[b, j // page_size], j % page_size], the key of every query head; its first dv elements are the value, its last
dr carry the rotary position. The reference keeps a contiguous cache of sequences of one length and rotates and normalises with
`mla_decode` and `div_softmax` (3-amd-mla-decode/amd-mla-submission.py:265-290); here every sequence has its own length and
position, read by the kernels on the device. The work is done by sm_100a CUDA kernels in lib/libb200fp8mm.so reached through the
C ABI of include/b200_mla_cache.h. There is no CPU path."""
from __future__ import annotations

import ctypes
import math

import torch

from . import _lib
from .fp8_mm import Fp8MmError, _check, _status, _status_words

_TYPES = {torch.bfloat16: 0, torch.float16: 1}


def _distinct(t):
    """No two elements of the tensor share an address."""
    need = 1
    for stride, size in sorted((st, sz) for st, sz in zip(t.stride(), t.shape) if sz > 1):
        if stride < need:
            return False
        need += stride * (size - 1)
    return True


def _apart(a, b):
    """No element of one tensor is an element of the other (two column ranges of the same rows are apart)."""
    if a.numel() == 0 or b.numel() == 0:
        return True
    (a0, a1), (b0, b1) = ((t.data_ptr(), t.data_ptr() + t.element_size() * (1 + sum(st * (sz - 1) for st, sz in zip(t.stride(), t.shape))))
                          for t in (a, b))
    if a1 <= b0 or b1 <= a0:
        return True
    if a.element_size() != b.element_size() or a.stride() != b.stride() or a.dim() < 2:
        return False
    pitch = math.gcd(*a.stride()[:-1]) * a.element_size()
    if pitch == 0:
        return False
    off = (b0 - a0) % pitch
    return a.shape[-1] * a.element_size() <= off and off + b.shape[-1] * b.element_size() <= pitch


def _same_or_apart(name_a, a, name_b, b):
    same = a.data_ptr() == b.data_ptr() and a.stride() == b.stride() and a.shape == b.shape
    _check(same or _apart(a, b), f"{name_b} must be {name_a} itself or lie apart from it")


def _check_cache(cache, block_table, lens, dv):
    """The checks that every entry point makes of the cache; (batch, capacity in slots)."""
    _check(cache.dim() == 3 and cache.dtype in _TYPES, "cache must be [pages, page_size, dv + dr] in bfloat16 or float16")
    pages, page_size, d = cache.shape
    _check(isinstance(dv, int) and dv % 128 == 0 and 128 <= dv <= 512, "dv must be 128, 256, 384 or 512")
    _check(dv <= d <= 576 and d % 64 == 0, "dr (the elements of a cache row behind dv) must be a multiple of 64, and dv + dr at most 576")
    _check(pages > 0 and page_size > 0, "cache must have pages and slots")
    _check(cache.stride(2) == 1 and cache.stride(0) % 8 == 0 and cache.stride(1) % 8 == 0 and cache.stride(0) >= d
           and cache.stride(1) >= d and cache.data_ptr() % 16 == 0,
           "cache rows must be contiguous, with strides that are multiples of 8 elements and a 16-byte aligned base")
    _check(block_table.dim() == 2 and block_table.dtype == torch.int32 and block_table.shape[1] > 0
           and block_table.stride(1) == 1, "block_table must be int32 [batch, pages per sequence] with contiguous rows")
    batch = block_table.shape[0]
    _check(batch < 65536, "at most 65535 sequences")
    _check(lens.dtype == torch.int32 and tuple(lens.shape) == (batch,) and (batch < 2 or lens.stride(0) == 1),
           "lens must be contiguous int32 [batch]")
    capacity = block_table.shape[1] * page_size
    _check(capacity <= 1 << 30, "at most 2**30 slots per sequence")
    return batch, capacity


def _check_slots(name, t, dtype, batch, capacity):
    """A value per slot of every sequence."""
    _check(t.dtype == dtype and t.dim() == 2 and t.shape[0] == batch and t.shape[1] >= capacity and t.stride(1) == 1,
           f"{name} must be {str(dtype).replace('torch.', '')} [batch, slots] with contiguous rows of at least {capacity} slots")


def _check_heads(name, t, cache, batch, width):
    _check(t.dtype == cache.dtype and t.dim() == 3 and t.shape[0] == batch and t.shape[1] > 0 and t.shape[2] == width
           and t.stride(2) == 1, f"{name} must be [batch, heads, {width}] in the cache's type with a contiguous last dimension")


def _check_device(*tensors):
    """All on one CUDA device, which is returned."""
    dev = tensors[0].device
    _check(all(t.is_cuda for t in tensors), "all tensors must be CUDA tensors (there is no CPU path)")
    _check(all(t.device == dev for t in tensors), "tensors on different devices")
    return dev


def _c_cache(cache, block_table, lens, dv):
    return _lib.CMlaCache(cache.data_ptr(), block_table.data_ptr(), lens.data_ptr(), _TYPES[cache.dtype], cache.shape[0],
                          cache.shape[1], dv, cache.shape[2] - dv, block_table.shape[0], block_table.shape[1],
                          cache.stride(0), cache.stride(1), block_table.stride(0))


def _ptr(t):
    return None if t is None else t.data_ptr()


def _workspace(dev, nbytes):
    """Scratch of one call. It comes from torch's allocator on the current stream, so calls on other streams and other
    captured graphs never share it."""
    return torch.empty(nbytes, dtype=torch.uint8, device=dev)


def mla_cache_append(row, position, cache, block_table, lens, dv: int, theta: float = 10000.0, q=None, q_out=None, score=None,
                     slot_position=None):
    """Writes one new row per sequence into the cache and rotates the queries for the same positions, on the current stream.

    row [batch, dv + dr] (what `kv_down_projection_fp8` returns) goes to slot lens[b] of sequence b, its last dr elements
    rotated for position[b] (int32 [batch]); block_table must name the slot's page already, and lens is not changed. A
    sequence whose lens[b] is negative or at the block table's capacity, or whose page is not one of the cache's, is left alone.
    No two sequences may name the same page for their new slots.
    q [batch, heads, dv + dr], optional: its last dr elements are rotated for the same positions into q_out (default: q itself;
    the others are copied). score (float32) and slot_position (int32), [batch, slots], optional: the new slot's entries become 0
    and position[b]. The rotation pairs element t with t + dr/2, angle position * theta**(-2t/dr), and unlike `mla_decode`
    neither rounds the angle nor the products to bf16: one rounding, at the end. Returns q_out."""
    if _lib.host_calls().mla_cache_append(row, position, cache, block_table, lens, dv, theta, q, q_out, score, slot_position):
        return q if q_out is None else q_out
    # Not the plain case, or a call that will be refused: the same checks here, with their errors.
    batch, capacity = _check_cache(cache, block_table, lens, dv)
    d = cache.shape[2]
    _check(_distinct(cache), "cache must not overlap itself")
    _check(row.dtype == cache.dtype and tuple(row.shape) == (batch, d) and row.stride(1) == 1,
           f"row must be [batch, {d}] in the cache's type with contiguous rows")
    _check(position.dtype == torch.int32 and tuple(position.shape) == (batch,) and (batch < 2 or position.stride(0) == 1),
           "position must be contiguous int32 [batch]")
    theta = float(theta)
    _check(theta > 0 and math.isfinite(theta), "theta must be positive and finite")
    tensors = [row, position, cache, block_table, lens]
    _check(q is not None or q_out is None, "q_out without q")
    _check(_apart(row, cache), "row must not lie in the cache")
    if q is not None:
        q_out = q if q_out is None else q_out
        _check_heads("q", q, cache, batch, d)
        _check_heads("q_out", q_out, cache, batch, d)
        _check(q.shape[1] == q_out.shape[1] and q.shape[1] <= 1 << 20, "q and q_out disagree on the heads, or have too many")
        _check(_distinct(q_out), "q_out must not overlap itself")
        _same_or_apart("q", q, "q_out", q_out)
        _check(_apart(q_out, row) and _apart(q_out, cache) and _apart(q, cache), "q, q_out, row and cache must lie apart")
        tensors += [q, q_out]
    for name, t, dtype in (("score", score, torch.float32), ("slot_position", slot_position, torch.int32)):
        if t is not None:
            _check_slots(name, t, dtype, batch, capacity)
            _check(_distinct(t), f"{name} must not overlap itself")
            tensors.append(t)
    dev = _check_device(*tensors)
    if batch == 0:
        return q_out
    with torch.cuda.device(dev):
        rc = _lib.load().b200_mla_cache_append(
            ctypes.byref(_c_cache(cache, block_table, lens, dv)), row.data_ptr(), row.stride(0), position.data_ptr(), theta,
            _ptr(q), *((q.stride(0), q.stride(1)) if q is not None else (0, 0)),
            _ptr(q_out), *((q_out.stride(0), q_out.stride(1)) if q is not None else (0, 0)),
            q.shape[1] if q is not None else 0,
            _ptr(score), score.stride(0) if score is not None else 0,
            _ptr(slot_position), slot_position.stride(0) if slot_position is not None else 0,
            torch.cuda.current_stream(dev).cuda_stream)
    if rc != 0:
        raise Fp8MmError(rc, "mla_cache_append")
    return q_out


def mla_cache_attend(q, cache, block_table, lens, dv: int, scale: float, out=None, score=None, score_out=None, max_len=None,
                     return_lse: bool = False):
    """Attention of one new token per sequence over its cached rows, on the current stream: out [batch, heads, dv], or
    (out, lse) with return_lse, lse float32 [batch, heads].

    out[b, h] = sum over j < lens[b] of p_j * row_j[:dv], p = softmax(scale * q[b, h] . row_j); q [batch, heads, dv + dr] carries
    the up-projection of the keys already. A sequence without rows gets zeros (lse -inf), and so does a head whose logits are all
    -inf (it adds nothing to the scores); what lies behind a sequence's last row is never looked at. lens above the block table's capacity count as the capacity; a page that is not one of the cache's reads
    as rows of zeros. score (float32 [batch, slots]), optional: score_out[b, j] = score[b, j] + the weights that slot j received
    from all heads (score_out default: score itself), j < lens[b]; other entries are left as they were. max_len, optional: no
    sequence is longer (longer ones are cut to it); it sizes the scratch that the weights need, batch * heads * max_len floats.

    Sums, maxima and joins are in 32 bits; the weights are rounded to the cache's type before they meet the values. A call repeats to
    the bit. Where a long sequence is split depends on the other sequences' lengths, and so does the order of its sums."""
    done = _lib.host_calls().mla_cache_attend(q, cache, block_table, lens, dv, scale, out, score, score_out, max_len, return_lse, _status)
    if done is not False:
        return done
    batch, capacity = _check_cache(cache, block_table, lens, dv)
    d = cache.shape[2]
    _check_heads("q", q, cache, batch, d)
    heads = q.shape[1]
    _check(heads <= 1 << 16, "at most 65536 heads")
    _check(all(size == 1 or (stride % 8 == 0 and stride >= d) for size, stride in zip(q.shape[:2], q.stride()))
           and q.data_ptr() % 16 == 0,
           "q: strides must be multiples of 8 elements, at least a row's, and the base address a multiple of 16 bytes")
    scale = float(scale)
    _check(abs(scale) < 2.0 ** 127, "scale must be finite and below 2**127 in magnitude")
    _check(max_len is None or (isinstance(max_len, int) and max_len > 0), "max_len must be a positive integer")
    max_len = capacity if max_len is None else min(max_len, capacity)
    tensors = [q, cache, block_table, lens]
    if out is None:
        out = torch.empty(batch, heads, dv, dtype=q.dtype, device=q.device)
    else:
        _check_heads("out", out, cache, batch, dv)
        _check(out.shape[1] == heads, "q and out disagree on the heads")
        _check(_distinct(out) and _apart(out, q) and _apart(out, cache), "out must not overlap itself, q or the cache")
    tensors.append(out)
    _check(score is not None or score_out is None, "score_out without score")
    if score is not None:
        score_out = score if score_out is None else score_out
        for name, t in (("score", score), ("score_out", score_out)):
            _check_slots(name, t, torch.float32, batch, capacity)
            tensors.append(t)
        _check(_distinct(score_out), "score_out must not overlap itself")
        _same_or_apart("score", score, "score_out", score_out)
    dev = _check_device(*tensors)
    lse = torch.empty(batch, heads, dtype=torch.float32, device=dev) if return_lse else None
    if batch > 0:
        lib = _lib.load()
        with torch.cuda.device(dev):
            ws = _workspace(dev, lib.b200_mla_cache_attend_workspace_bytes(batch, heads, dv, d - dv, max_len, score is not None))
            rc = lib.b200_mla_cache_attend(
                ctypes.byref(_c_cache(cache, block_table, lens, dv)), q.data_ptr(), q.stride(0), q.stride(1), heads, scale,
                out.data_ptr(), out.stride(0), out.stride(1), _ptr(lse),
                _ptr(score), score.stride(0) if score is not None else 0,
                _ptr(score_out), score_out.stride(0) if score is not None else 0,
                max_len, ws.data_ptr(), ws.numel(), _status_words(dev).data_ptr(),
                torch.cuda.current_stream(dev).cuda_stream)
        if rc != 0:
            raise Fp8MmError(rc, "mla_cache_attend")
    return (out, lse) if return_lse else out


def selftest_wait_expiry(device="cuda", heads: int = 16, page_size: int = 16, limit_ms: float = 5.0):
    """Diagnostics: makes waits inside the attention's kernel run out on purpose, in the allowed way. A sequence of four tiles is attended
    to with every wait limited to `limit_ms` and the second tile's copy left out; the kernel gives up, returns by itself and reports the
    wait. Returns the four status words [code, wait, block, phase]; code 1 is WAIT_EXPIRED. The words are cleared again."""
    dev = torch.device(device)
    if dev.index is None:
        dev = torch.device("cuda", torch.cuda.current_device())
    lib, dv, d = _lib.load(), 512, 576
    with torch.cuda.device(dev):
        rows = 192
        pages = -(-rows // page_size)
        cache = torch.zeros(pages, page_size, d, dtype=torch.bfloat16, device=dev)
        table = torch.arange(pages, dtype=torch.int32, device=dev)[None]
        lens = torch.full((1,), rows, dtype=torch.int32, device=dev)
        q, out = (torch.zeros(1, heads, width, dtype=torch.bfloat16, device=dev) for width in (d, dv))
        ws = _workspace(dev, lib.b200_mla_cache_attend_workspace_bytes(1, heads, dv, d - dv, table.shape[1] * page_size, 0))
        st = _status_words(dev)
        torch.cuda.synchronize(dev)
        rc = lib.b200_mla_cache_attend_selftest_wait_expiry(
            ctypes.byref(_c_cache(cache, table, lens, dv)), q.data_ptr(), q.stride(0), q.stride(1), heads, 1.0, out.data_ptr(),
            out.stride(0), out.stride(1), ws.data_ptr(), ws.numel(), int(limit_ms * 1e6), 1, st.data_ptr(),
            torch.cuda.current_stream(dev).cuda_stream)
        if rc != 0:
            raise Fp8MmError(rc, "selftest_wait_expiry")
        torch.cuda.synchronize(dev)
        words = st.tolist()
        st.zero_()
        torch.cuda.synchronize(dev)
    return words


def mla_cache_evict(cache, block_table, lens, score, slot_position, budget: int, recent: int, lens_out=None, score_out=None,
                    position_out=None):
    """Shortens every sequence of more than `budget` rows to `budget`, on the current stream; returns lens_out.

    Kept are the rows whose slot_position (int32 [batch, slots]) is above the sequence's largest minus `recent`, then those of
    the largest score (float32 [batch, slots]; the lower slot first among equals, NaN above every number), `budget` in all. Kept
    rows in slots at or behind the budget move, in ascending order, to the slots below it that were given up: rows inside the
    cache, scores and positions into score_out and position_out, of which the slots below the new length are written. lens_out,
    score_out and position_out default to the inputs themselves. Slots are in no particular order afterwards, which no
    attention over rotated rows can tell; what lies behind the budget is left as it was, and its pages are free. A page with
    slots below the budget must belong to one sequence alone."""
    lens_out = lens if lens_out is None else lens_out
    score_out = score if score_out is None else score_out
    position_out = slot_position if position_out is None else position_out
    if _lib.host_calls().mla_cache_evict(cache, block_table, lens, score, slot_position, budget, recent, lens_out, score_out, position_out):
        return lens_out
    batch, capacity = _check_cache(cache, block_table, lens, dv=128)
    _check(_distinct(cache), "cache must not overlap itself")
    _check(isinstance(budget, int) and isinstance(recent, int) and 0 < budget < 1 << 31 and 0 <= recent <= budget,
           "budget must be positive and recent between 0 and budget")
    _check(lens_out.dtype == torch.int32 and tuple(lens_out.shape) == (batch,) and (batch < 2 or lens_out.stride(0) == 1),
           "lens_out must be contiguous int32 [batch]")
    for name, t, dtype in (("score", score, torch.float32), ("slot_position", slot_position, torch.int32),
                           ("score_out", score_out, torch.float32), ("position_out", position_out, torch.int32)):
        _check_slots(name, t, dtype, batch, capacity)
    _check(_distinct(score_out) and _distinct(position_out), "score_out and position_out must not overlap themselves")
    _same_or_apart("lens", lens, "lens_out", lens_out)
    _same_or_apart("score", score, "score_out", score_out)
    _same_or_apart("slot_position", slot_position, "position_out", position_out)
    dev = _check_device(cache, block_table, lens, score, slot_position, lens_out, score_out, position_out)
    if batch == 0:
        return lens_out
    lib = _lib.load()
    with torch.cuda.device(dev):
        ws = _workspace(dev, lib.b200_mla_cache_evict_workspace_bytes(batch, capacity, budget))
        rc = lib.b200_mla_cache_evict(
            ctypes.byref(_c_cache(cache, block_table, lens, 128)), score.data_ptr(), score.stride(0), slot_position.data_ptr(),
            slot_position.stride(0), budget, recent, lens_out.data_ptr(), score_out.data_ptr(), score_out.stride(0),
            position_out.data_ptr(), position_out.stride(0), ws.data_ptr(), ws.numel(),
            torch.cuda.current_stream(dev).cuda_stream)
    if rc != 0:
        raise Fp8MmError(rc, "mla_cache_evict")
    return lens_out
