"""CPU: what the paged-cache operators and the sampler refuse, and how work over ragged batches is cut (host arithmetic, no GPU)."""
import ctypes as C

import pytest

from spy_b200 import backend as B

P = 1 << 20   # an aligned address that nothing reads


def cache(**k):
    c = B.paged_cache(P, P, 8, 16, 2, k.pop("head_dim", 64))
    for n, v in k.items():
        setattr(c, n, v)
    return c


def batch(**k):
    b = B.paged_batch(P, P, P, 3, 7, 4)
    for n, v in k.items():
        setattr(b, n, v)
    return b


def attention(c=None, b=None, n_head=4, **k):
    d = B.paged_attention_desc(c or cache(), b or batch(), P, P, n_head)
    for n, v in k.items():
        setattr(d, n, v)
    return d


def append(c=None, b=None, n_head=4, **k):
    d = B.paged_append_desc(c or cache(), b or batch(), P, P, P, P, n_head)
    for n, v in k.items():
        setattr(d, n, v)
    return d


def sample(**k):
    d = B.sample_desc(P, B.FP32, 4, 1000, P, uniform=P)
    for n, v in k.items():
        setattr(d, n, v)
    return d


@pytest.mark.parametrize("d", [
    attention(), append(), sample(), attention(window=5), attention(causal=0), attention(out_type=B.FP32), append(rope_mode=B.ROPE_NONE, rope_dim=0),
    append(n_head=0, q=None, q_out=None), append(in_type=B.FP16), sample(number_type=B.FP16, uniform=None), sample(n_rows=0), attention(b=batch(n_seq=0, row_start=None, n_kv=None)),
    attention(b=batch(table_stride=0, page_table=None)), append(c=cache(head_dim=256)), attention(n_head=6, scale=0.25), sample(n_rows=1, row_stride=0), sample(n_vocab=1 << 20, row_stride=1 << 20),
])
def test_taken(d):
    assert B.refusal(d) == ""


@pytest.mark.parametrize("word,d", [
    ("type", attention(c=cache(number_type=B.FP32))), ("aligned", attention(c=cache(k=P + 8))), ("aligned", attention(c=cache(v=None))), ("pages", attention(c=cache(n_pages=0))),
    ("pages", attention(c=cache(page_size=0))), ("heads", attention(c=cache(n_head_kv=0))), ("strides", attention(c=cache(token_stride=68))), ("strides", attention(c=cache(page_stride=-8))),
    ("heads of 72", attention(c=cache(head_dim=72))), ("heads of 256", attention(c=cache(head_dim=256))), ("elements", append(c=cache(head_dim=264))), ("elements", append(c=cache(head_dim=12))),
    ("sequences", attention(b=batch(n_seq=-1))), ("rows", attention(b=batch(n_rows=-2))), ("rows", attention(b=batch(max_rows=-1))), ("row_start", attention(b=batch(row_start=None))),
    ("n_kv", append(b=batch(n_kv=None))), ("page_table", append(b=batch(page_table=None))), ("aligned", append(b=batch(n_kv=P + 2))), ("query heads", attention(n_head=5)),
    ("query heads", attention(n_head=0)), ("aligned", attention(q=None)), ("aligned", attention(out=P + 4)), ("16 bytes", attention(q_stride=260)), ("16 bytes", attention(out_stride=258, out_type=B.FP32)),
    ("output of type", attention(out_type=B.Q8_0)), ("window", attention(window=-1)), ("window", attention(window=4, causal=0)), ("scale", attention(scale=float("inf"))), ("scale", attention(scale=float("nan"))),
    ("type", append(in_type=B.INT32)), ("type", append(q_out_type=B.Q4_0)), ("query heads", append(q=None)), ("query heads", append(n_head=0)), ("aligned", append(q_out=None)), ("aligned", append(k=P + 4)),
    ("16 bytes", append(v_stride=130)), ("16 bytes", append(in_type=B.FP16, k_stride=132)), ("mode", append(rope_mode=1)), ("rotated", append(rope_dim=0)), ("rotated", append(rope_dim=72)),
    ("rotated", append(rope_dim=20)), ("base", append(freq_base=0.0)), ("base", append(freq_base=float("inf"))), ("scale", append(freq_scale=float("nan"))),
    ("type", sample(number_type=B.Q8_0)), ("logits", sample(n_rows=-1)), ("logits", sample(n_vocab=0)), ("logits", sample(n_vocab=(1 << 20) + 1, row_stride=1 << 21)), ("apart", sample(row_stride=999)),
    ("there", sample(logits=None)), ("there", sample(ids=None)), ("aligned", sample(probs=P + 2)), ("aligned", sample(top_k=P + 1)), ("aligned", sample(logits=P + 2)),
])
def test_refused(word, d):
    assert word in B.refusal(d)


def test_a_message_without_room_is_left_out():
    lib = B.lib()
    assert lib.spyb_sample_check(C.byref(sample(n_vocab=0)), None, 0) == B.UNSUPPORTED
    assert lib.spyb_sample_check(None, None, 0) == B.FAIL
    buf = C.create_string_buffer(b"xxxxxxxx", 8)
    assert lib.spyb_sample_check(C.byref(sample(n_vocab=0)), buf, 4) == B.UNSUPPORTED and buf.raw[3:] == b"\0xxxx" and buf.value == b"sam"


def test_no_backend_no_call():
    lib = B.lib()
    assert lib.spyb_paged_attention(None, C.byref(attention())) == B.FAIL
    assert lib.spyb_paged_append(None, C.byref(append())) == B.FAIL
    assert lib.spyb_sample(None, C.byref(sample())) == B.FAIL


def test_pieces_cover_every_item_once():
    """The CTAs' stretches of a ragged batch, on lengths that make sense and on ones that do not (negative, beyond the tables, not ascending)."""
    assert B.lib().spyb_selftest_host() == 0
