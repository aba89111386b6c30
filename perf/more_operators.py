"""Caches of 8 bits, norms of queries and keys, and batches that share a beginning: the paged operators that go beyond ``perf/operators.py``.

``store``   ``B200Backend.paged_store``: new tokens' Q and K are normalised head by head and rotated to their positions, K and V go to the cache pages of their sequences in
            fp16, or as 8-bit integers with a scale for each head of each position; these are read back by ``B200Backend.paged_load``, as values
``load``    ``B200Backend.paged_load``: K and V of whole sequences out of 8-bit pages, as contiguous fp16 rows
``attend``  ``B200Backend.paged_attend``: attention over 8-bit pages, and over pages whose beginning several sequences share

Widths are those of LLaMa2-7B and 13B, the architectures of this repository's configurations, or shared K/V heads beside the same number of query heads. Pages are handed
out in random order and hold stale values where nothing was stored yet.
"""
import math

import torch

own = False

MOST_FLOPS, MOST_BYTES = 2.5e11, 6.0e8          # of a drawn case; the listed ones have up to 2.58e11 and 6.4e8


def _attend(name, rows, kv, n_head, n_head_kv, head_dim=128, page=16, window=0, layout="head", cache="int8", groups="", shared="0"):
    """rows / kv: new tokens and positions of the sequences: "16x1" is sixteen of one; "a..b" is spread between a and b. groups: numbers of sequences side by side that share
    their first `shared` positions ("3x8": three groups of eight), which come in front of kv's."""
    return dict(op="attend", name=name, rows=rows, kv=kv, n_head=n_head, n_head_kv=n_head_kv, head_dim=head_dim, page=page, window=window, layout=layout, cache=cache, groups=groups,
                shared=shared)


def _store(name, rows, kv, n_head, n_head_kv, head_dim=128, page=16, mode=0, rope_dim=128, base=10000.0, dtype="f32", layout="head", cache="int8"):
    return dict(op="store", name=name, rows=rows, kv=kv, n_head=n_head, n_head_kv=n_head_kv, head_dim=head_dim, page=page, mode=mode, rope_dim=rope_dim, base=base, dtype=dtype,
                layout=layout, cache=cache)


def _load(name, kv, n_head_kv, head_dim=128, page=16, layout="head"):
    return dict(op="load", name=name, rows=kv, kv=kv, n_head_kv=n_head_kv, head_dim=head_dim, page=page, layout=layout, cache="int8")


def listed():
    return [
        # a single conversation's next token, shared K/V heads: the smallest call, where the launches are all
        _store("store 1 token 32+8, int8", "1x1", "1x41", 32, 8),
        # a step of ninety-six running requests, far into long contexts, fp16 pages; pairs as halves, as most models with normalised queries and keys have them
        _store("store 96 sequences 40+8, fp16", "96x1", "96x50..120000", 40, 8, mode=2, base=1000000.0, cache="fp16"),
        # the prompts of five requests, in odd lengths and pages
        _store("store prompts 40+8, int8", "5x1100..2500", "5x2600..2900", 40, 8, page=24, mode=2, layout="token"),
        # a short conversation leaves the card; then six long ones, for another server with other pages
        _load("load 1 of 300, 8 heads", "1x300", 8),
        _load("load 6 to 24000, 8 heads", "6x9000..24000", 8, page=64, layout="token"),
        # the next token at the end of a 7B conversation of four thousand: few heads' worth of work for a whole chip
        _attend("decode 1 at 4000, 32+32, int8", "1x1", "1x4001", 32, 32),
        # sixty-four requests of all lengths up to 4096
        _attend("decode 64 to 4096, 32+8, int8", "64x1", "64x30..4096", 32, 8),
        # three long documents
        _attend("decode 3 at 100000, 40+8, int8", "3x1", "3x90000..110000", 40, 8, page=64, layout="token"),
        # five guessed tokens a request, checked in one pass
        _attend("verify 5 of 24 to 9000, 32+8, int8", "24x5", "24x100..9000", 32, 8),
        # a prompt's chunk beside the running requests of the same step
        _attend("chunk 1500 + 24 decodes, 40+8, int8", "1x1500,24x1", "1x9111,24x200..6000", 40, 8, page=32),
        # sixty-four requests behind one long system prompt
        _attend("decode 64 behind 6000, 32+8, fp16", "64x1", "64x5..600", 32, 8, cache="fp16", groups="1x64", shared="6000"),
        # guessed tokens of four users' agents, each with its own documents, in 8 bits
        _attend("verify 3 of 4 x 12 behind 2000..16000, 40+8, int8", "48x3", "48x40..900", 40, 8, page=32, groups="4x12", shared="4x2000..16000"),
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def _draw_heads(rng):
    n_kv = rng.choice([1, 2, 4, 5, 8, 16])
    return n_kv * rng.choice([1, 2, 3, 4, 5, 7, 8] if n_kv < 16 else [1, 2]), n_kv


def _draw(rng):
    op = rng.choice(["store", "store", "load", "attend", "attend", "attend", "attend"])
    n_head, n_kv = _draw_heads(rng)
    some = dict(op=op, n_head_kv=n_kv, head_dim=rng.choice([64, 128, 128]), page=rng.choice([8, 16, 16, 24, 32, 64, 128]), layout=rng.choice(["head", "token"]))
    hd = some["head_dim"]
    if op == "load":
        most = _log(rng, 20, 30000)
        kv = f"{_log(rng, 1, 40)}x{max(1, most // 4)}..{most}"
        return dict(some, rows=kv, kv=kv, cache="int8")
    some["n_head"] = n_head
    together = op == "attend" and rng.random() < 0.5            # batches that share something
    kind = rng.choice(["decode", "decode", "verify", "chunk", "mixed"]) if not together else rng.choice(["decode", "verify"])
    n_seq = _log(rng, 1, 100) if kind in ("decode", "verify") else _log(rng, 1, 8)
    past = _log(rng, 64, 60000 if kind in ("decode", "verify") else 12000)
    group = [_log(rng, 1, 6), _log(rng, 2, 40)]
    if together:
        n_seq, past = group[0] * group[1], _log(rng, 12, 2000)
    if kind == "decode":
        rows, kv = f"{n_seq}x1", f"{n_seq}x{max(2, past // 8)}..{past}"
    elif kind == "verify":
        rows, kv = f"{n_seq}x{rng.randint(2, 9)}", f"{n_seq}x{max(10, past // 8)}..{past + 10}"
    else:
        chunk = _log(rng, 16, 2600)
        rows, kv = f"{n_seq}x{max(1, chunk // 2)}..{chunk}", f"{n_seq}x{rng.choice([0, past // 2])}..{past}"
        if kind == "mixed":
            more = _log(rng, 1, 40)
            rows, kv = rows + f",{more}x1", kv + f",{more}x{max(2, past // 8)}..{past}"
    if op == "store":
        return dict(some, rows=rows, kv=kv, mode=rng.choice([0, 2]), rope_dim=rng.choice([hd, hd, hd // 2]), base=rng.choice([10000.0, 500000.0, 1000000.0]),
                    dtype=rng.choice(["f32", "f32", "f16"]), cache=rng.choice(["int8", "int8", "fp16"]))
    if together:
        most = _log(rng, 150, 20000)
        return dict(some, rows=rows, kv=kv, window=0, cache=rng.choice(["int8", "fp16"]), groups=f"{group[0]}x{group[1]}", shared=f"{group[0]}x{max(1, most // 2)}..{most}")
    return dict(some, rows=rows, kv=kv, window=rng.choice([0, 0, 0, _log(rng, 32, 4096)]), cache="int8", groups="", shared="0")


def draw(rng):
    while True:
        case = _draw(rng)
        w, (rows, kv, _, _) = work(case), _lengths(case)
        if w["bytes"] <= MOST_BYTES and w["flops"] <= MOST_FLOPS and sum(kv) * case["n_head_kv"] * case["head_dim"] <= 3.2e8 \
                and max(r * k for r, k in zip(rows, kv)) * case.get("n_head", 1) <= 6e8:      # (stale parts of the pools and the plain form's score rows stay in bounds too)
            return case


# ---------------------------------------------------------------------------------------------- lengths
def _spread(text):
    """"3x5,2x10..20": numbers of a list, those between two bounds a fixed odd stride apart."""
    got = []
    for part in text.split(","):
        n, v = part.split("x") if "x" in part else ("1", part)
        lo, hi = (int(t) for t in (v.split("..") if ".." in v else (v, v)))
        got += [lo + (i * 7919 + 13) * 104729 % max(1, hi - lo + 1) if hi > lo else lo for i in range(int(n))]
    return got


def _lengths(case):
    """New tokens and positions of every sequence, how many sequences a group has, and what it shares."""
    rows = _spread(case["rows"])
    kv = [max(r, k) for r, k in zip(rows, _spread(case["kv"]))]
    groups = _spread(case["groups"]) if case.get("groups") else [1] * len(rows)
    groups = [n for n in groups if n > 0]
    shared = _spread(case["shared"]) if case.get("groups") else [0]
    shared = (shared * len(groups))[:len(groups)]
    first = 0
    for n, common in zip(groups, shared):
        kv[first:first + n] = [k + common for k in kv[first:first + n]]
        first += n
    return rows, kv, groups, shared


# ---------------------------------------------------------------------------------------------- 8 bits
def _scale_of(most):
    """The smallest fp16 that is not below most / 127."""
    exact = most / 127
    near = exact.half()
    return torch.where(near.to(exact.dtype) < exact, (near.view(torch.int16) + 1).view(torch.float16), near)


def _to_8_bits(x):
    """x: [..., head_dim] in 32 bits or more. Integers and their heads' scales."""
    scale = _scale_of(x.abs().amax(-1))
    wide = scale.to(x.dtype)[..., None]
    return torch.where(wide > 0, torch.round(x / wide), torch.zeros_like(x)).to(torch.int8), scale


# ---------------------------------------------------------------------------------------------- states
class _State:
    desc = None


def _paged(case, seed):
    """Pools with stale values in them, pages in random order, lengths as device arrays beside the host's."""
    s = _State()
    s.case, s.op = case, case["op"]
    gen = s.gen = torch.Generator(device="cuda").manual_seed(seed)
    s.rows, s.kv, s.groups, s.shared = _lengths(case)
    page, h_kv, hd = case["page"], case["n_head_kv"], case["head_dim"]
    need = [-(-n // page) for n in s.kv]
    common, first = [0] * len(need), 0                      # whole pages that a sequence has from the first one of its group
    leads = list(range(len(need)))
    for n, shared in zip(s.groups, s.shared):
        for i in range(first + 1, first + n):
            common[i], leads[i] = shared // page, first
        first += n
    s.n_pages, s.width = sum(need) - sum(common) + 3, max(need)
    order = torch.randperm(s.n_pages, generator=gen, device="cuda").int()
    s.table = torch.full((len(need), s.width), -1, dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(need):
        s.table[i, :common[i]] = s.table[leads[i], :common[i]]
        s.table[i, common[i]:n] = order[at:at + n - common[i]]
        at += n - common[i]
    shape = (s.n_pages, h_kv, page, hd) if case["layout"] == "head" else (s.n_pages, page, h_kv, hd)
    s.k_pool = torch.randn(shape, generator=gen, device="cuda", dtype=torch.float16)
    s.v_pool = torch.randn(shape, generator=gen, device="cuda", dtype=torch.float16)
    if case["cache"] == "int8":
        # values as heads of a projection have them: some positions and heads larger than others
        s.scales = torch.empty(shape[:3] + (2,), device="cuda", dtype=torch.float16)
        for i, name in enumerate(("k_pool", "v_pool")):
            pool = getattr(s, name)
            size = torch.exp(0.5 * torch.randn(shape[:3], generator=gen, device="cuda"))
            integers = torch.empty(shape, device="cuda", dtype=torch.int8)
            for a in range(0, s.n_pages, 4096):
                integers[a:a + 4096], s.scales[a:a + 4096, ..., i] = _to_8_bits(pool[a:a + 4096].float() * size[a:a + 4096, ..., None])
            setattr(s, name, integers)
    for i, (n, shared) in enumerate(zip(s.groups, s.shared)):   # the last page that is shared in part: the same values in pages of their own
        tail = shared % page
        if tail and n > 1:
            lead = sum(s.groups[:i])
            pages = s.table[lead:lead + n, shared // page].long()
            for pool in (s.k_pool, s.v_pool) + ((s.scales,) if case["cache"] == "int8" else ()):
                view = pool if case["layout"] == "token" else pool.transpose(1, 2)
                view[pages[1:], :tail] = view[pages[0], :tail].clone()
    starts = torch.tensor([0] + s.rows).cumsum(0).int()
    s.n_rows = int(starts[-1])
    s.row_start, s.n_kv = starts.cuda(), torch.tensor(s.kv, dtype=torch.int32).cuda()
    return s


def _paged_views(s):
    """The pools, and where there are any the scales, as [page][position][head][...]."""
    pools = (s.k_pool, s.v_pool) + ((s.scales,) if s.case["cache"] == "int8" else ())
    return pools if s.case["layout"] == "token" else tuple(p.transpose(1, 2) for p in pools)


def prepare(case, seed):
    s = _paged(case, seed)
    h_kv, hd = case["n_head_kv"], case["head_dim"]
    if case["op"] == "store":
        h = case["n_head"]
        # Q, K and V side by side, as one projection leaves them
        s.qkv = torch.randn((s.n_rows, (h + 2 * h_kv) * hd), generator=s.gen, device="cuda", dtype=torch.float16 if case["dtype"] == "f16" else torch.float32)
        s.q_norm, s.k_norm = 1 + 0.3 * torch.randn((2, hd), generator=s.gen, device="cuda")
        s.q_out = torch.zeros((s.n_rows, h, hd), device="cuda", dtype=torch.float16)
    if case["op"] == "attend":
        h = case["n_head"]
        sharp = 0.5 + 2.5 * torch.rand((1, h, 1), generator=s.gen, device="cuda")       # some heads look at few positions, some at all
        s.q = (sharp * torch.randn((s.n_rows, h, hd), generator=s.gen, device="cuda")).half()
        s.out = torch.empty_like(s.q)
        s.group_start = torch.tensor([0] + s.groups).cumsum(0).int().cuda()
        s.n_shared = torch.tensor(s.shared, dtype=torch.int32).cuda()
    elif case["cache"] == "int8":
        s.k_out, s.v_out = (torch.empty((s.n_rows, h_kv, hd), device="cuda", dtype=torch.float16) for _ in range(2))
    return s


# ---------------------------------------------------------------------------------------------- the framework's calls
_kept = []


def _backend():
    if not _kept:
        from spy_b200 import backend
        _kept.append(backend.B200Backend(0))
    return _kept[0]


def _describe(s):
    """The descriptors that a program keeps beside its buffers."""
    from spy_b200 import backend as B
    case, hd, h_kv = s.case, s.case["head_dim"], s.case["n_head_kv"]
    token_major, eight = case["layout"] == "token", case["cache"] == "int8"
    cache = B.paged_cache(s.k_pool.data_ptr(), s.v_pool.data_ptr(), s.n_pages, case["page"], h_kv, hd, token_major=token_major, number_type=B.INT8 if eight else B.FP16)
    scales = B.paged_scales(s.scales.data_ptr(), case["page"], h_kv, token_major=token_major) if eight else None
    batch = B.paged_batch(s.row_start.data_ptr(), s.n_kv.data_ptr(), s.table.data_ptr(), len(s.rows), s.n_rows, s.width, max_rows=max(s.rows))
    if s.op == "attend":
        attention = B.paged_attention_desc(cache, batch, s.q.data_ptr(), s.out.data_ptr(), case["n_head"], window=case["window"])
        if not case["groups"]:
            return [B.paged_attend_desc(attention, scales)]
        size = B.paged_attend_workspace(len(s.rows), s.n_rows, case["n_head"], hd)
        s.workspace = torch.empty(size, dtype=torch.uint8, device="cuda")
        return [B.paged_attend_desc(attention, scales, group_start=s.group_start.data_ptr(), n_shared=s.n_shared.data_ptr(), n_group=len(s.groups), workspace=s.workspace.data_ptr(),
                                    workspace_bytes=size)]
    load = [B.paged_load_desc(cache, batch, s.k_out.data_ptr(), s.v_out.data_ptr(), scales)] if eight else []
    if s.op == "load":
        return load
    h, size = case["n_head"], s.qkv.element_size() * hd
    append = B.paged_append_desc(cache, batch, s.qkv.data_ptr(), s.qkv.data_ptr() + h * size, s.qkv.data_ptr() + (h + h_kv) * size, s.q_out.data_ptr(), h,
                                 in_type=B.FP16 if case["dtype"] == "f16" else B.FP32, row_stride=(h + 2 * h_kv) * hd, rope_mode=case["mode"], rope_dim=case["rope_dim"],
                                 freq_base=case["base"])
    return [B.paged_store_desc(append, scales, q_norm=s.q_norm.data_ptr(), k_norm=s.k_norm.data_ptr(), norm_eps=1e-6)] + load


def _own(s):
    if s.desc is None:
        s.desc = _describe(s)
    if s.op == "attend":
        _backend().paged_attend(s.desc[0])
        return s.out
    if s.op == "load":
        _backend().paged_load(s.desc[0])
        return {"k": s.k_out, "v": s.v_out}
    _backend().paged_store(s.desc[0])
    if s.case["cache"] == "fp16":
        return {"q": s.q_out, "k": s.k_pool, "v": s.v_pool}
    _backend().paged_load(s.desc[1])
    return {"q": s.q_out, "k": s.k_out, "v": s.v_out}


# ---------------------------------------------------------------------------------------------- plain forms
def _places(s):
    """Page and position in it of every row, and the position in its sequence."""
    row = torch.arange(s.n_rows, device="cuda")
    seq = torch.searchsorted(s.row_start, row, right=True) - 1
    pos = s.n_kv[seq] - s.row_start[seq + 1] + row
    return s.table[seq, pos // s.case["page"]].long(), (pos % s.case["page"]).long(), pos


def _plain_load(s, page, slot):
    views = _paged_views(s)
    scales = views[2][page, slot].float()
    s.k_out.copy_((views[0][page, slot].float() * scales[..., 0:1]).half())
    s.v_out.copy_((views[1][page, slot].float() * scales[..., 1:2]).half())
    return {"k": s.k_out, "v": s.v_out}


def _plain_store(s):
    case, hd, rot = s.case, s.case["head_dim"], s.case["rope_dim"]
    h, h_kv = case["n_head"], case["n_head_kv"]
    page, slot, pos = _places(s)
    pair = torch.arange(rot // 2, device="cuda", dtype=torch.float64)
    angle = (pos.double()[:, None] * torch.pow(torch.tensor(case["base"], dtype=torch.float64, device="cuda"), -2 * pair / rot))[:, None, :]
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    a = torch.arange(0, rot, 2, device="cuda") if case["mode"] == 0 else torch.arange(rot // 2, device="cuda")
    b = a + 1 if case["mode"] == 0 else a + rot // 2
    x = s.qkv.view(s.n_rows, h + 2 * h_kv, hd).float()
    qk = x[:, :h + h_kv]
    qk = qk * torch.rsqrt((qk * qk).mean(-1, keepdim=True) + 1e-6)
    qk = torch.cat([qk[:, :h] * s.q_norm, qk[:, h:] * s.k_norm], 1)
    turned = qk.clone()
    turned[:, :, a] = qk[:, :, a] * cos - qk[:, :, b] * sin
    turned[:, :, b] = qk[:, :, a] * sin + qk[:, :, b] * cos
    s.q_out.copy_(turned[:, :h].half())
    k, v, views = turned[:, h:], x[:, h + h_kv:], _paged_views(s)
    if case["cache"] == "fp16":
        views[0][page, slot] = k.half()
        views[1][page, slot] = v.half()
        return {"q": s.q_out, "k": s.k_pool, "v": s.v_pool}
    k8, k_scale = _to_8_bits(k)
    v8, v_scale = _to_8_bits(v)
    views[0][page, slot] = k8
    views[1][page, slot] = v8
    views[2][page, slot] = torch.stack([k_scale, v_scale], -1)
    return dict(_plain_load(s, page, slot), q=s.q_out)


def _plain_attend(s):
    case, hd, h, h_kv = s.case, s.case["head_dim"], s.case["n_head"], s.case["n_head_kv"]
    views = _paged_views(s)
    alike = {}
    for i, n in enumerate(s.rows):                          # sequences with the same number of new tokens go together, padded to the longest
        alike.setdefault(n, []).append(i)
    for n, seqs in alike.items():
        longest = max(s.kv[i] for i in seqs)
        which = torch.tensor(seqs, device="cuda")
        pos = torch.arange(longest, device="cuda")
        page, slot = s.table[which][:, pos // case["page"]].clamp(min=0).long(), pos % case["page"]
        k, v = (x[page, slot].permute(0, 2, 1, 3).float() for x in views[:2])                      # [sequence][head][position][element]
        if case["cache"] == "int8":
            scales = views[2][page, slot].permute(0, 2, 1, 3).float()
            k *= scales[..., 0:1]
            v *= scales[..., 1:2]
        rows = s.row_start[which].long()[:, None] + torch.arange(n, device="cuda")
        q = s.q[rows].float().view(len(seqs), n, h_kv, h // h_kv, hd).permute(0, 2, 3, 1, 4).reshape(len(seqs), h_kv, -1, hd)
        at = s.n_kv[which][:, None] - n + torch.arange(n, device="cuda")                          # [sequence][row]
        seen = pos <= at[:, :, None]
        if case["window"]:
            seen &= pos > at[:, :, None] - case["window"]
        scores = torch.matmul(q, k.transpose(2, 3)).mul_(1 / math.sqrt(hd)).view(len(seqs), h_kv, h // h_kv, n, longest)
        scores.masked_fill_(~seen[:, None, None], -math.inf)
        p = scores.sub_(scores.amax(-1, keepdim=True)).exp_()
        total = p.sum(-1, keepdim=True)
        out = torch.matmul(p.view(len(seqs), h_kv, -1, longest), v).view(len(seqs), h_kv, h // h_kv, n, hd) / total
        s.out[rows] = out.permute(0, 3, 1, 2, 4).reshape(len(seqs), n, h, hd).half()
    return s.out


def run(state):
    if own:
        return _own(state)
    if state.op == "load":
        page, slot, _ = _places(state)
        return _plain_load(state, page, slot)
    return _plain_store(state) if state.op == "store" else _plain_attend(state)


# ---------------------------------------------------------------------------------------------- by the definition, in 64 bits
def _exact_load(s):
    views, first = _paged_views(s), 0
    k, v = (torch.empty((s.n_rows,) + views[0].shape[2:], dtype=torch.float64, device="cuda") for _ in range(2))
    for i, (n, kv) in enumerate(zip(s.rows, s.kv)):
        pages = s.table[i, :-(-kv // s.case["page"])].long()
        integers = [x[pages].flatten(0, 1)[kv - n:kv].double() for x in views]
        k[first:first + n] = integers[0] * integers[2][..., :1]
        v[first:first + n] = integers[1] * integers[2][..., 1:]
        first += n
    return {"k": k, "v": v}


def _exact_store(s):
    case, hd, rot, h, h_kv = s.case, s.case["head_dim"], s.case["rope_dim"], s.case["n_head"], s.case["n_head_kv"]
    eight = case["cache"] == "int8"
    pools = None if eight else [s.k_pool.double(), s.v_pool.double()]
    views = None if eight else pools if case["layout"] == "token" else [p.transpose(1, 2) for p in pools]
    got = {"q": torch.empty((s.n_rows, h, hd), dtype=torch.float64, device="cuda")}
    if eight:
        got.update({n: torch.empty((s.n_rows, h_kv, hd), dtype=torch.float64, device="cuda") for n in ("k", "v")})
    else:
        got.update(k=pools[0], v=pools[1])
    speeds = torch.tensor([case["base"] ** (-2.0 * i / rot) for i in range(rot // 2)], dtype=torch.float64, device="cuda")
    weights = torch.cat([s.q_norm.double().expand(h, hd), s.k_norm.double().expand(h_kv, hd)])
    first = 0
    for i, (n, kv) in enumerate(zip(s.rows, s.kv)):
        x = s.qkv[first:first + n].double().view(n, h + 2 * h_kv, hd)
        qk = x[:, :h + h_kv] / torch.sqrt(torch.linalg.vector_norm(x[:, :h + h_kv], dim=-1, keepdim=True) ** 2 / hd + 1e-6) * weights
        where = torch.arange(kv - n, kv, device="cuda")
        turn = torch.polar(torch.ones((n, rot // 2), dtype=torch.float64, device="cuda"), where.double()[:, None] * speeds)[:, None]
        head = qk[:, :, :rot]
        pairs = head.reshape(n, -1, rot // 2, 2) if case["mode"] == 0 else torch.stack([head[..., :rot // 2], head[..., rot // 2:]], -1)
        turned = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
        turned = turned.reshape(n, -1, rot) if case["mode"] == 0 else torch.cat([turned[..., 0], turned[..., 1]], -1)
        full = torch.cat([turned, qk[:, :, rot:]], -1)
        got["q"][first:first + n] = full[:, :h]
        for name, y in (("k", full[:, h:]), ("v", x[:, h + h_kv:])):
            if eight:
                unit = y.abs().amax(-1, keepdim=True) / 127
                step = unit.half()                              # (the next one up where that is below)
                step = torch.where(step.double() < unit, torch.nextafter(step, torch.full_like(step, math.inf)), step).double()
                got[name][first:first + n] = torch.where(step > 0, torch.round(y / step) * step, torch.zeros_like(y))
            else:
                views[0 if name == "k" else 1][s.table[i][where // case["page"]].long(), where % case["page"]] = y
        first += n
    return got


def _exact_attend(s):
    case, hd, h, h_kv = s.case, s.case["head_dim"], s.case["n_head"], s.case["n_head_kv"]
    views = _paged_views(s)
    out = torch.empty((s.n_rows, h, hd), dtype=torch.float64, device="cuda")
    first = 0
    for i, (n, kv) in enumerate(zip(s.rows, s.kv)):
        pages = s.table[i, :-(-kv // case["page"])].long()
        held = [x[pages].flatten(0, 1)[:kv] for x in views]                                   # [position][head][element]
        block = max(1, int(2e8) // (kv * (h // h_kv)))
        for g in range(h_kv):
            kg, vg = held[0][:, g].double(), held[1][:, g].double()
            if case["cache"] == "int8":
                kg, vg = kg * held[2][:, g, :1].double(), vg * held[2][:, g, 1:].double()
            for r in range(0, n, block):
                m = min(block, n - r)
                q = s.q[first + r:first + r + m, g * (h // h_kv):(g + 1) * (h // h_kv)].double()
                t = torch.einsum("rhe,pe->rhp", q, kg) / hd ** 0.5
                ago = (kv - n + r + torch.arange(m, device="cuda"))[:, None] - torch.arange(kv, device="cuda")[None]
                hidden = (ago < 0) | (ago >= case["window"]) if case["window"] else ago < 0
                t = t.masked_fill(hidden[:, None], -math.inf)
                out[first + r:first + r + m, g * (h // h_kv):(g + 1) * (h // h_kv)] = torch.einsum("rhp,pe->rhe", torch.exp(t - torch.logsumexp(t, -1, keepdim=True)), vg)
        first += n
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return {"store": _exact_store, "load": _exact_load, "attend": _exact_attend}[case["op"]](s)


# ---------------------------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    rows, kv, groups, shared = _lengths(case)
    h_kv, hd, n = case["n_head_kv"], case["head_dim"], sum(rows)
    eight = case["cache"] == "int8"
    cell = 2 * h_kv * (hd + 2 if eight else 2 * hd)            # K and V of a position as they are kept
    if case["op"] == "load":
        return {"bytes": n * (cell + 4 * h_kv * hd), "flops": 2 * n * h_kv * hd}
    h = case["n_head"]
    if case["op"] == "store":
        size = 2 if case["dtype"] == "f16" else 4
        return {"bytes": n * ((h + 2 * h_kv) * hd * size + 2 * h * hd + cell + (4 * h_kv * hd if eight else 0)), "flops": n * (4 * (h + h_kv) * hd + 3 * (h + h_kv) * case["rope_dim"])}
    reach = case["window"] or 1 << 40
    read = sum(min(k, r + reach - 1) for r, k in zip(rows, kv)) - sum((g - 1) * c for g, c in zip(groups, shared))   # positions that some row sees, what is shared once
    pairs = 0
    for r, k in zip(rows, kv):                                                 # row i sees min(k - r + i + 1, reach) positions
        full = max(0, min(r, reach - (k - r)))                                 # rows that see their whole past
        pairs += full * (k - r) + full * (full + 1) // 2 + (r - full) * reach if reach < 1 << 40 else r * (k - r) + r * (r + 1) // 2
    return {"bytes": 4 * n * h * hd + read * cell, "flops": 4 * pairs * h * hd}
