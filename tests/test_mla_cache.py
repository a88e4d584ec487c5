"""Refusals of the paged-cache operators. They are checked before anything touches a GPU, so CPU tensors show them; a call that
passes every other check is refused for being on the CPU."""
import os
import re

import pytest
import torch

import amd_developer_challenge_2025_b200 as pkg

B, H, DV, D, PS, PER = 3, 5, 128, 192, 16, 4


def base():
    z = torch.zeros
    return dict(
        cache=z(20, PS, D, dtype=torch.bfloat16), block_table=z(B, PER, dtype=torch.int32), lens=z(B, dtype=torch.int32),
        q=z(B, H, D, dtype=torch.bfloat16), row=z(B, D, dtype=torch.bfloat16), position=z(B, dtype=torch.int32),
        score=z(B, PS * PER), slot_position=z(B, PS * PER, dtype=torch.int32))


def append(t, dv=DV, **more):
    return pkg.mla_cache_append(t["row"], t["position"], t["cache"], t["block_table"], t["lens"], dv, q=t["q"],
                                score=t["score"], slot_position=t["slot_position"], **more)


def attend(t, dv=DV, scale=0.1, **more):
    return pkg.mla_cache_attend(t["q"], t["cache"], t["block_table"], t["lens"], dv, scale, score=t["score"], **more)


def evict(t, budget=8, recent=2, **more):
    return pkg.mla_cache_evict(t["cache"], t["block_table"], t["lens"], t["score"], t["slot_position"], budget, recent, **more)


CALLS = {"append": append, "attend": attend, "evict": evict}


@pytest.mark.parametrize("call", CALLS)
def test_cpu_tensors(call):
    with pytest.raises(ValueError, match="CUDA"):
        CALLS[call](base())


@pytest.mark.parametrize("call", CALLS)
@pytest.mark.parametrize("name,bad,match", [
    ("cache", lambda t: t.float(), "cache must be"),
    ("cache", lambda t: t[0], "cache must be"),
    ("cache", lambda t: t[:0], "pages and slots"),
    ("cache", lambda t: t[:, :0], "pages and slots"),
    ("cache", lambda t: t[:, :, :190], "dr"),
    ("cache", lambda t: torch.zeros(20, PS, 640, dtype=t.dtype), "dr"),
    ("cache", lambda t: torch.zeros(20, PS, D + 4, dtype=t.dtype)[:, :, :D], "strides"),
    ("cache", lambda t: torch.zeros(20, PS, D + 8, dtype=t.dtype)[:, :, 1:D + 1], "aligned"),
    ("cache", lambda t: torch.zeros(20, D, PS, dtype=t.dtype).transpose(1, 2), "contiguous"),
    ("cache", lambda t: t[:1].expand(20, PS, D), "strides"),
    ("block_table", lambda t: t.long(), "block_table"),
    ("block_table", lambda t: t[0], "block_table"),
    ("block_table", lambda t: t[:, :0], "block_table"),
    ("block_table", lambda t: torch.zeros(PER, B, dtype=t.dtype).t(), "block_table"),
    ("lens", lambda t: t.long(), "lens"),
    ("lens", lambda t: t[:2], "lens"),
    ("lens", lambda t: torch.zeros(2 * B, dtype=t.dtype)[::2], "lens"),
])
def test_bad_caches(call, name, bad, match):
    t = base()
    t[name] = bad(t[name])
    with pytest.raises(ValueError, match=match):
        CALLS[call](t)


@pytest.mark.parametrize("call", ["append", "attend"])
@pytest.mark.parametrize("dv", [0, 64, 130, 256, 640, 128.0])
def test_bad_dv(call, dv):
    with pytest.raises(ValueError, match="d[vr]"):
        CALLS[call](base(), dv=dv)


@pytest.mark.parametrize("name,bad,match", [
    ("row", lambda t: t[:2], "row must"), ("row", lambda t: t.half(), "row must"), ("row", lambda t: t[:, :128], "row must"),
    ("position", lambda t: t.long(), "position"), ("position", lambda t: t[:1], "position"),
    ("q", lambda t: t.half(), "q must"), ("q", lambda t: t[:, :0], "q must"), ("q", lambda t: t[:2], "q must"),
    ("q", lambda t: t[:, :1].expand(B, H, D), "overlap itself"),
    ("score", lambda t: t.double(), "score must"), ("score", lambda t: t[:, :-1], "score must"),
    ("slot_position", lambda t: t.float(), "slot_position must"),
    ("slot_position", lambda t: t[:1].expand(B, PS * PER), "overlap itself"),
])
def test_bad_append(name, bad, match):
    t = base()
    t[name] = bad(t[name])
    with pytest.raises(ValueError, match=match):
        append(t)


def test_append_arguments_that_disagree():
    t = base()
    for theta in (0.0, -1.0, float("inf"), float("nan")):
        with pytest.raises(ValueError, match="theta"):
            append(t, theta=theta)
    with pytest.raises(ValueError, match="heads"):
        append(t, q_out=torch.zeros(B, H + 1, D, dtype=torch.bfloat16))
    wide = torch.zeros(B, H + 1, D, dtype=torch.bfloat16)
    t["q"] = wide[:, :H]
    with pytest.raises(ValueError, match="itself or lie apart"):
        append(t, q_out=wide[:, 1:])
    t = base()
    t["row"] = t["cache"][0, :B]
    with pytest.raises(ValueError, match="row must not lie in the cache"):
        append(t)
    t = base()
    t["q"] = None
    with pytest.raises(ValueError, match="q_out without q"):
        append(t, q_out=wide)


@pytest.mark.parametrize("name,bad,match", [
    ("q", lambda t: t.float(), "q must"), ("q", lambda t: t[..., :128], "q must"), ("q", lambda t: t[:, :0], "q must"),
    ("q", lambda t: torch.zeros(B, H, D + 4, dtype=t.dtype)[..., :D], "multiples of 8"),
    ("q", lambda t: torch.zeros(B, H, D + 8, dtype=t.dtype)[..., 4:D + 4], "16 bytes"),
    ("score", lambda t: t.half(), "score must"), ("score", lambda t: t[:, :-1], "score must"),
])
def test_bad_attend(name, bad, match):
    t = base()
    t[name] = bad(t[name])
    with pytest.raises(ValueError, match=match):
        attend(t)


def test_attend_arguments_that_disagree():
    t = base()
    for scale in (float("inf"), float("nan"), 1e300, -3e38):
        with pytest.raises(ValueError, match="scale"):
            attend(t, scale=scale)
    for max_len in (0, -1, 2.5):
        with pytest.raises(ValueError, match="max_len"):
            attend(t, max_len=max_len)
    with pytest.raises(ValueError, match="heads"):
        attend(t, out=torch.zeros(B, H - 1, DV, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="out must"):
        attend(t, out=torch.zeros(B, H, DV))
    with pytest.raises(ValueError, match="overlap"):
        attend(t, out=t["q"][..., :DV])
    with pytest.raises(ValueError, match="itself or lie apart"):
        flat = torch.zeros(B * PS * PER + 1)
        t["score"] = flat[:-1].view(B, -1)
        attend(t, score_out=flat[1:].view(B, -1))
    t["score"] = None
    with pytest.raises(ValueError, match="score_out without score"):
        attend(t, score_out=torch.zeros(B, PS * PER))


def test_column_ranges_of_the_same_rows_are_apart():
    """The output may lie behind the query in one buffer, and the score behind another score."""
    t = base()
    wide = torch.zeros(B, H, D + DV, dtype=torch.bfloat16)
    t["q"] = wide[..., :D]
    scores = torch.zeros(B, 2 * PS * PER)
    t["score"] = scores[:, :PS * PER]
    with pytest.raises(ValueError, match="CUDA"):
        attend(t, out=wide[..., D:], score_out=scores[:, PS * PER:])


@pytest.mark.parametrize("budget,recent", [(0, 0), (-1, 0), (8, 9), (8, -1), (8.0, 1), (1 << 31, 1)])
def test_bad_budgets(budget, recent):
    with pytest.raises(ValueError, match="budget"):
        evict(base(), budget, recent)


def test_evict_outputs_that_do_not_fit():
    t = base()
    for name, bad, match in (("lens_out", torch.zeros(B), "lens_out"), ("lens_out", torch.zeros(B + 1, dtype=torch.int32), "lens_out"),
                             ("score_out", torch.zeros(B, PS), "score_out"),
                             ("score_out", torch.zeros(1, PS * PER).expand(B, -1), "overlap themselves"),
                             ("position_out", torch.zeros(B, PS * PER), "position_out")):
        with pytest.raises(ValueError, match=match):
            evict(t, **{name: bad})


def test_error_codes_without_launch(built_library):
    """The C entry points check for themselves."""
    import ctypes

    from amd_developer_challenge_2025_b200 import _lib

    lib = _lib.load()
    one = 4096  # never dereferenced: every check below fails first

    def cache(**change):
        c = _lib.CMlaCache(one, one, one, 0, 20, PS, DV, D - DV, B, PER, PS * D, D, PER)
        for k, v in change.items():
            setattr(c, k, v)
        return ctypes.byref(c)

    def call(c, q=one, heads=H, scale=0.1, q_sb=H * D, ws=one, ws_bytes=1 << 30):
        return lib.b200_mla_cache_attend(c, q, q_sb, D, heads, scale, one, H * DV, DV, None, None, 0, None, 0, 0, ws, ws_bytes, None, None)

    assert call(None) == 1 and call(cache(data=None)) == 1 and call(cache(lens=None)) == 1 and call(cache(), q=None) == 1
    for change in (dict(dtype=2), dict(batch=0), dict(batch=65536), dict(pages=0), dict(page_size=0), dict(pages_per_seq=0),
                   dict(dv=64), dict(dv=640), dict(dr=32), dict(dr=-64), dict(dr=512), dict(page_size=1 << 30)):
        assert call(cache(**change)) == 2, change
    assert call(cache(), heads=0) == 2 and call(cache(), scale=float("nan")) == 2 and call(cache(), scale=3e38) == 2
    assert call(cache(slot_stride=D - 8)) == 3 and call(cache(page_stride=PS * D + 4)) == 3 and call(cache(), q_sb=H * D + 1) == 3
    assert call(cache(data=4100)) == 4 and call(cache(), q=4104) == 4
    assert call(cache(), ws=None) == 6 and call(cache(), ws_bytes=0) == 6 and call(cache(), ws=4100) == 6
    assert lib.b200_mla_cache_attend_workspace_bytes(0, H, DV, D - DV, 64, 0) == 0

    def put(c, row=one, theta=1e4, q=None, q_out=None, heads=0):
        return lib.b200_mla_cache_append(c, row, D, one, theta, q, 0, 0, q_out, 0, 0, heads, None, 0, None, 0, None)

    assert put(None) == 1 and put(cache(), row=None) == 1 and put(cache(), q=one) == 1
    assert put(cache(), theta=0.0) == 2 and put(cache(), q=one, q_out=one, heads=0) == 2 and put(cache(data=4100)) == 4

    def drop(c, budget=8, recent=2, score=one, ws=one, ws_bytes=1 << 30):
        return lib.b200_mla_cache_evict(c, score, 64, one, 64, budget, recent, one, one, 64, one, 64, ws, ws_bytes, None)

    assert drop(None) == 1 and drop(cache(), score=None) == 1
    assert drop(cache(), budget=0) == 2 and drop(cache(), recent=9) == 2 and drop(cache(), recent=-1) == 2
    assert drop(cache(), ws=None) == 6 and drop(cache(), ws_bytes=0) == 6
    assert lib.b200_mla_cache_evict_workspace_bytes(B, 0, 8) == 0


def test_no_read_only_loads():
    """The kernels begin under the kernel before them, which may still write what they read: nothing may go through the read-only path."""
    with open(os.path.join(os.path.dirname(pkg.__file__), "csrc", "mla_cache_sm100.cu")) as f:
        code = re.sub(r"//[^\n]*", "", f.read())
    assert "griddepcontrol.wait" in code
    for form in (r"__ldg\s*\(", r"\bld\.global\.nc", r"\bconst\s+[\w:]+\s*\*\s*__restrict__"):
        assert not re.search(form, code), form


def test_error_codes_of_the_wait_self_test(built_library):
    import ctypes

    from amd_developer_challenge_2025_b200 import _lib

    lib, one = _lib.load(), 4096  # never dereferenced

    def call(limit=5000000, skip=1, status=one, ws=None):
        c = _lib.CMlaCache(one, one, one, 0, 20, PS, DV, D - DV, B, PER, PS * D, D, PER)
        return lib.b200_mla_cache_attend_selftest_wait_expiry(ctypes.byref(c), one, H * D, D, H, 1.0, one, H * DV, DV, ws, 1 << 30, limit, skip,
                                                              status, None)

    assert call(status=None) == 1 and call(skip=-1) == 2 and call() == 6
    assert call(limit=999999) == call(limit=100000001) == call(limit=0) == 7


def test_plans_ask_the_device_for_its_sms():
    """No rule takes a number of SMs as given; where there is no device, sizes are worked out for a B200."""
    with open(os.path.join(os.path.dirname(pkg.__file__), "csrc", "mla_cache_sm100.cu")) as f:
        code = re.sub(r"//[^\n]*", "", f.read())
    assert re.findall(r"[^\n]*\b148\b[^\n]*", code) == ["constexpr int kSmsOfB200 = 148;"]
