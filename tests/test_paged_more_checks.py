"""CPU: what storing with norms and in bytes, reading back and attention over shared beginnings refuse."""
import ctypes as C

import pytest

from spy_b200 import backend as B

P = 1 << 20   # an aligned address that nothing reads
BIG = 1 << 40


def cache(number_type=B.INT8, head_dim=64, **k):
    c = B.paged_cache(P, P, 8, 16, 2, head_dim, number_type=number_type)
    for n, v in k.items():
        setattr(c, n, v)
    return c


def scales(**k):
    s = B.paged_scales(P, 16, 2)
    for n, v in k.items():
        setattr(s, n, v)
    return s


def batch(**k):
    b = B.paged_batch(P, P, P, 3, 7, 4)
    for n, v in k.items():
        setattr(b, n, v)
    return b


def with_fields(d, k):
    for n, v in k.items():
        setattr(d, n, v)
    return d


def store(c=None, s=None, b=None, n_head=4, q=P, **k):
    d = B.paged_append_desc(c or cache(), b or batch(), q if n_head else None, P, P, P if n_head else None, n_head)
    own = {n: k.pop(n) for n in ("q_norm", "k_norm", "norm_eps") if n in k}
    return B.paged_store_desc(with_fields(d, k), s or scales(), **own)


def load(c=None, s=None, b=None, **k):
    return with_fields(B.paged_load_desc(c or cache(), b or batch(), P, P, s or scales()), k)


def attend(c=None, s=None, b=None, n_head=4, groups=None, **k):
    return B.paged_attend_desc(with_fields(B.paged_attention_desc(c or cache(), b or batch(), P, P, n_head), k), s or scales(), **(groups or {}))


def groups(**k):
    return dict(dict(group_start=P, n_shared=P, n_group=2, workspace=P, workspace_bytes=BIG), **k)


FP16 = cache(B.FP16)


@pytest.mark.parametrize("d", [
    store(), store(q_norm=P, k_norm=P, norm_eps=1e-5), store(c=FP16, s=B.PagedScales()), store(n_head=0), store(n_head=0, k_norm=P), store(rope_mode=B.ROPE_NONE, rope_dim=0), store(in_type=B.FP16),
    store(c=cache(head_dim=256)), store(s=scales(page_stride=0, token_stride=0, head_stride=0)), load(), load(c=FP16, s=B.PagedScales()), load(out_type=B.FP32), load(k=None), load(v=None, v_stride=3),
    attend(), attend(c=FP16, s=B.PagedScales()), attend(window=9), attend(groups=groups()), attend(groups=groups(), window=9), attend(groups=groups(), causal=0), attend(c=cache(head_dim=96)),
    attend(b=batch(n_seq=0, n_rows=0, row_start=None, n_kv=None), groups=groups(workspace=None, workspace_bytes=0)), attend(groups=groups(n_group=0, group_start=None, n_shared=None, workspace=None)),
    attend(groups=groups(workspace_bytes=B.paged_attend_workspace(3, 7, 4, 64))), attend(c=FP16, groups=groups()),
])
def test_taken(d):
    assert B.refusal(d) == ""


@pytest.mark.parametrize("word,d", [
    ("paged_store: a cache of type 0 (fp16 or int8", store(c=cache(B.FP32))), ("paged_store: the scales", store(s=B.PagedScales())), ("scales", store(s=scales(pairs=P + 2))), ("scales", store(s=scales(token_stride=-1))),
    ("multiples of 16 elements", store(c=cache(token_stride=72))), ("multiples of 16 elements", store(c=cache(head_dim=24))), ("multiples of 8 elements", store(c=cache(B.FP16, token_stride=68))),
    ("norms", store(q_norm=P + 4)), ("norms", store(k_norm=P + 8)), ("norms", store(n_head=0, q_norm=P)), ("norm_eps", store(norm_eps=-1e-9)), ("norm_eps", store(norm_eps=float("nan"))),
    ("norm_eps", store(norm_eps=float("inf"))), ("paged_store: q, k, v", store(k=None)), ("paged_store: rope mode", store(rope_mode=7)), ("paged_store: 72 rotated", store(rope_dim=72)),
    ("query heads", store(q=None)), ("n_kv", store(b=batch(n_kv=None))), ("paged_store: row strides", store(v_stride=130)),
    ("paged_load: a cache", load(c=cache(B.Q8_0))), ("scales", load(s=B.PagedScales())), ("k or v", load(k=None, v=None)), ("k or v", load(k=P + 8)), ("output of type", load(out_type=B.INT8)),
    ("strides", load(k_stride=129)), ("strides", load(out_type=B.FP32, v_stride=130)), ("rows", load(b=batch(n_rows=-1))), ("aligned", load(c=cache(v=P + 8))),
    ("paged_attend: a cache of type 0", attend(c=cache(B.FP32))), ("scales", attend(s=B.PagedScales())), ("paged_attend: heads of 72", attend(c=cache(B.FP16, head_dim=72))),
    ("paged_attend: 5 query heads", attend(n_head=5)), ("paged_attend: a window", attend(window=3, causal=0)), ("paged_attend: scale", attend(scale=float("nan"))), ("paged_attend: q and out", attend(q=None)),
    ("output of type", attend(out_type=B.INT8)), ("groups", attend(groups=groups(n_group=-1))), ("groups", attend(groups=groups(n_group=1 << 24))), ("group_start", attend(groups=groups(group_start=None))),
    ("group_start", attend(groups=groups(n_shared=P + 2))), ("workspace", attend(groups=groups(workspace=None))), ("workspace", attend(groups=groups(workspace=P + 8))),
    ("workspace", attend(groups=groups(workspace_bytes=B.paged_attend_workspace(3, 7, 4, 64) - 1))),
])
def test_refused(word, d):
    assert word in B.refusal(d)


def test_the_fp16_operators_take_no_bytes():
    assert "type 24" in B.refusal(B.paged_attention_desc(cache(), batch(), P, P, 4)) and "type 24" in B.refusal(B.paged_append_desc(cache(), batch(), P, P, P, P, 4))


def test_room_for_two_passes():
    """Accumulators, two statistics and two words of who has them a row and head, four words a sequence; nothing where a size makes no sense."""
    n = B.paged_attend_workspace(3, 7, 4, 64)
    assert 7 * 4 * (64 * 4 + 16) + 4 * 3 * 4 <= n <= 7 * 4 * (64 * 4 + 16) + 4 * 3 * 4 + 32
    assert B.paged_attend_workspace(-1, 7, 4, 64) == B.paged_attend_workspace(1, 1 << 24, 4, 64) == B.paged_attend_workspace(1, 7, -4, 64) == 0
    assert B.paged_attend_workspace(1, (1 << 24) - 1, 128, 128) > 1 << 40


def test_no_backend_no_call():
    lib = B.lib()
    assert lib.spyb_paged_store(None, C.byref(store())) == lib.spyb_paged_load(None, C.byref(load())) == lib.spyb_paged_attend(None, C.byref(attend())) == B.FAIL
    assert lib.spyb_paged_store_check(None, None, 0) == lib.spyb_paged_load_check(None, None, 0) == lib.spyb_paged_attend_check(None, None, 0) == B.FAIL
