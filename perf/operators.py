"""The operators of a server step over paged caches, over the ranges that its users meet.

``append``     ``B200Backend.paged_append``: the new tokens' Q and K are rotated to their positions, K and V go to the cache pages of
               their sequences;
``attention``  ``B200Backend.paged_attention``: the new tokens of every sequence (one, a few, a chunk of a prompt) attend to its pages;
``sample``     ``B200Backend.sample``: the next token of every row of logits, from given uniform numbers.

Widths are those of LLaMa2-7B and 13B, the architectures of this repository's configurations, or shared K/V heads beside the same
number of query heads. Pages are handed out in random order and hold stale values where nothing was stored yet.
"""
import math

import numpy as np
import torch

own = False

MOST_FLOPS, MOST_BYTES = 2.5e11, 1.2e9          # of a drawn case; the listed ones have up to 2.58e11 and 1.22e9


def _attention(name, rows, kv, n_head, n_head_kv, head_dim=128, page=16, window=0, layout="head"):
    """rows / kv: new tokens and positions of the sequences: "16x1" is sixteen of one; "a..b" is spread between a and b."""
    return dict(op="attention", name=name, rows=rows, kv=kv, n_head=n_head, n_head_kv=n_head_kv, head_dim=head_dim, page=page, window=window, layout=layout)


def _append(name, rows, kv, n_head, n_head_kv, head_dim=128, page=16, mode=0, rope_dim=128, base=10000.0, dtype="f32", layout="head"):
    return dict(op="append", name=name, rows=rows, kv=kv, n_head=n_head, n_head_kv=n_head_kv, head_dim=head_dim, page=page, mode=mode, rope_dim=rope_dim,
                base=base, dtype=dtype, layout=layout)


def listed():
    return [
        # a single conversation's next token at 7B widths: the smallest call, where the launch is all
        _append("append 1 token 32+32", "1x1", "1x41", 32, 32),
        # a step of ninety-six running requests with shared K/V heads, far into long contexts; pairs as halves, as most models outside LLaMa's own files have them
        _append("append 96 sequences 40+8", "96x1", "96x50..120000", 40, 8, mode=2, base=500000.0),
        # the prompts of five requests at 13B widths, in odd lengths and pages
        _append("append prompts 40+40", "5x1100..2500", "5x2600..2900", 40, 40, page=24, layout="token"),
        # the next token at the end of a 7B conversation of four thousand: few heads' worth of work for a whole chip
        _attention("decode 1 at 4000, 32+32", "1x1", "1x4001", 32, 32),
        # sixty-four requests of all lengths up to 4096
        _attention("decode 64 to 4096, 32+8", "64x1", "64x30..4096", 32, 8),
        # three long documents
        _attention("decode 3 at 100000, 40+8", "3x1", "3x90000..110000", 40, 8, page=64, layout="token"),
        # five guessed tokens a request, checked in one pass
        _attention("verify 5 of 24 to 9000, 32+8", "24x5", "24x100..9000", 32, 8),
        # a prompt's last chunk of 512 tokens at 7B widths, context 4096
        _attention("chunk 512 at 3968, 32+32", "1x512", "1x3968", 32, 32),
        # a prompt's chunk beside the running requests of the same step
        _attention("chunk 1500 + 24 decodes, 40+8", "1x1500,24x1", "1x9111,24x200..6000", 40, 8, page=32),
        # whole prompts under a sliding window, narrow heads
        _attention("prompts 6 x 2000, window 1024, 32+4 x 64", "6x1500..2600", "6x0", 32, 4, head_dim=64, page=64, window=1024),
        # one reply's next token; then a full house, each request with settings of its own
        dict(op="sample", name="sample 1 of 32000", rows=1, vocab=32000, spread=2.5, settings="all"),
        dict(op="sample", name="sample 192 of 128000", rows=192, vocab=128000, spread=2.5, settings="mixed"),
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def _draw_heads(rng):
    n_kv = rng.choice([1, 2, 4, 5, 8, 16])
    return n_kv * rng.choice([1, 2, 3, 4, 5, 7, 8] if n_kv < 16 else [1, 2]), n_kv


def _draw(rng):
    op = rng.choice(["append", "attention", "attention", "attention", "sample"])
    if op == "sample":
        return dict(op=op, rows=_log(rng, 1, 190), vocab=_log(rng, 2000, 128000), spread=rng.choice([1.0, 2.5, 4.0]), settings=rng.choice(["mixed", "mixed", "all", "plain", "greedy"]))
    n_head, n_kv = _draw_heads(rng)
    head_dim = rng.choice([64, 128, 128])
    page, layout = rng.choice([8, 16, 16, 24, 32, 64, 128]), rng.choice(["head", "token"])
    kind = rng.choice(["decode", "decode", "verify", "chunk", "mixed"])
    n_seq = _log(rng, 1, 100) if kind in ("decode", "verify") else _log(rng, 1, 8)
    past = _log(rng, 64, 60000 if kind in ("decode", "verify") else 12000)
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
    if op == "append":
        mode = rng.choice([0, 2])
        return dict(op=op, rows=rows, kv=kv, n_head=n_head, n_head_kv=n_kv, head_dim=head_dim, page=page, mode=mode, rope_dim=rng.choice([head_dim, head_dim, head_dim // 2]),
                    base=rng.choice([10000.0, 500000.0, 1000000.0]), dtype=rng.choice(["f32", "f32", "f16"]), layout=layout)
    return dict(op=op, rows=rows, kv=kv, n_head=n_head, n_head_kv=n_kv, head_dim=head_dim, page=page, window=rng.choice([0, 0, 0, _log(rng, 32, 4096)]), layout=layout)


def draw(rng):
    while True:
        case = _draw(rng)
        if case["op"] == "sample":
            return case
        w, (rows, kv) = work(case), _lengths(case)
        if w["bytes"] <= MOST_BYTES and w["flops"] <= MOST_FLOPS and sum(kv) * case["n_head_kv"] * case["head_dim"] <= 3.2e8 \
                and max(r * k for r, k in zip(rows, kv)) * case["n_head"] <= 6e8:      # (stale parts of the pools and the plain form's score rows stay in bounds too)
            return case


# ---------------------------------------------------------------------------------------------- lengths
def _spread(text):
    """"3x5,2x10..20": numbers of a list, those between two bounds a fixed odd stride apart."""
    got = []
    for part in text.split(","):
        n, v = part.split("x")
        lo, hi = (int(t) for t in (v.split("..") if ".." in v else (v, v)))
        got += [lo + (i * 7919 + 13) * 104729 % max(1, hi - lo + 1) if hi > lo else lo for i in range(int(n))]
    return got


def _lengths(case):
    rows = _spread(case["rows"])
    return rows, [max(r, k) for r, k in zip(rows, _spread(case["kv"]))]


# ---------------------------------------------------------------------------------------------- states
class _State:
    desc = None


def _paged(case, seed):
    """Pools with stale values in them, pages in random order, lengths as device arrays beside the host's."""
    s = _State()
    s.case, s.op = case, case["op"]
    gen = s.gen = torch.Generator(device="cuda").manual_seed(seed)
    s.rows, s.kv = _lengths(case)
    page, h_kv, hd = case["page"], case["n_head_kv"], case["head_dim"]
    need = [-(-n // page) for n in s.kv]
    s.n_pages, s.width = sum(need) + 3, max(need)
    order = torch.randperm(s.n_pages, generator=gen, device="cuda").int()
    s.table = torch.full((len(need), s.width), -1, dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(need):
        s.table[i, :n] = order[at:at + n]
        at += n
    shape = (s.n_pages, h_kv, page, hd) if case["layout"] == "head" else (s.n_pages, page, h_kv, hd)
    s.k_pool = torch.randn(shape, generator=gen, device="cuda", dtype=torch.float16)
    s.v_pool = torch.randn(shape, generator=gen, device="cuda", dtype=torch.float16)
    starts = np.concatenate([[0], np.cumsum(s.rows)]).astype(np.int32)
    s.n_rows = int(starts[-1])
    s.row_start, s.n_kv = torch.from_numpy(starts).cuda(), torch.tensor(s.kv, dtype=torch.int32).cuda()
    return s


def _paged_views(s):
    """The pools as [page][position][head][element]."""
    return (s.k_pool, s.v_pool) if s.case["layout"] == "token" else (s.k_pool.transpose(1, 2), s.v_pool.transpose(1, 2))


def prepare(case, seed):
    if case["op"] == "sample":
        s = _State()
        s.case, s.op = case, "sample"
        gen = torch.Generator(device="cuda").manual_seed(seed)
        n, v = case["rows"], case["vocab"]
        uniform = lambda lo, hi: lo + (hi - lo) * torch.rand(n, generator=gen, device="cuda")  # noqa: E731
        # a broad background and some hundred likely tokens, as a language model's head gives them
        s.logits = case["spread"] * torch.randn((n, v), generator=gen, device="cuda") - 4
        likely = torch.randint(0, v, (n, min(v, 200)), generator=gen, device="cuda")
        s.logits.scatter_add_(1, likely, 6 * torch.rand(likely.shape, generator=gen, device="cuda") + 4)
        s.temperature, s.top_p, s.min_p, s.uniform = uniform(0.6, 1.3), uniform(0.7, 0.99), uniform(0.01, 0.1), uniform(0, 1).clamp_(max=1 - 2.0 ** -24)
        s.top_k = torch.randint(1, 101, (n,), generator=gen, device="cuda", dtype=torch.int32)
        row = torch.arange(n, device="cuda")
        if case["settings"] == "plain":                    # temperature alone
            s.top_k.zero_(), s.top_p.fill_(1), s.min_p.zero_()
        elif case["settings"] == "greedy":
            s.temperature.zero_()
        elif case["settings"] == "mixed":                  # each request leaves something out
            s.temperature[row % 8 == 3] = 0
            s.top_k[row % 2 == 1] = 0
            s.top_p[row % 3 == 1] = 1
            s.min_p[row % 5 != 2] = 0
        return s
    s = _paged(case, seed)
    h, h_kv, hd = case["n_head"], case["n_head_kv"], case["head_dim"]
    if case["op"] == "append":
        # Q, K and V side by side, as one projection leaves them
        s.qkv = torch.randn((s.n_rows, (h + 2 * h_kv) * hd), generator=s.gen, device="cuda", dtype=torch.float16 if case["dtype"] == "f16" else torch.float32)
        s.q_out = torch.zeros((s.n_rows, h, hd), device="cuda", dtype=torch.float16)
    else:
        sharp = 0.5 + 2.5 * torch.rand((1, h, 1), generator=s.gen, device="cuda")       # some heads look at few positions, some at all
        s.q = (sharp * torch.randn((s.n_rows, h, hd), generator=s.gen, device="cuda")).half()
        s.out = torch.empty_like(s.q)
    return s


# ---------------------------------------------------------------------------------------------- the framework's calls
_shared = []


def _backend():
    if not _shared:
        from spy_b200 import backend
        _shared.append(backend.B200Backend(0))
    return _shared[0]


def _describe(s):
    """The descriptor that a program keeps beside its buffers."""
    from spy_b200 import backend as B
    case = s.case
    if s.op == "sample":
        return B.sample_desc(s.logits.data_ptr(), B.FP32, case["rows"], case["vocab"], s.ids.data_ptr(), uniform=s.uniform.data_ptr(), temperature=s.temperature.data_ptr(),
                             top_k=s.top_k.data_ptr(), top_p=s.top_p.data_ptr(), min_p=s.min_p.data_ptr(), probs=s.probs.data_ptr())
    cache = B.paged_cache(s.k_pool.data_ptr(), s.v_pool.data_ptr(), s.n_pages, case["page"], case["n_head_kv"], case["head_dim"], token_major=case["layout"] == "token")
    batch = B.paged_batch(s.row_start.data_ptr(), s.n_kv.data_ptr(), s.table.data_ptr(), len(s.rows), s.n_rows, s.width, max_rows=max(s.rows))
    h, h_kv, hd = case["n_head"], case["n_head_kv"], case["head_dim"]
    if s.op == "attention":
        return B.paged_attention_desc(cache, batch, s.q.data_ptr(), s.out.data_ptr(), h, window=case["window"])
    size = s.qkv.element_size() * hd
    return B.paged_append_desc(cache, batch, s.qkv.data_ptr(), s.qkv.data_ptr() + h * size, s.qkv.data_ptr() + (h + h_kv) * size, s.q_out.data_ptr(), h,
                               in_type=B.FP16 if case["dtype"] == "f16" else B.FP32, row_stride=(h + 2 * h_kv) * hd, rope_mode=case["mode"], rope_dim=case["rope_dim"],
                               freq_base=case["base"])


def _own(s):
    if s.desc is None:
        if s.op == "sample":
            s.ids = torch.empty(s.case["rows"], dtype=torch.int32, device="cuda")
            s.probs = torch.empty(s.case["rows"], device="cuda")
        s.desc = _describe(s)
    if s.op == "append":
        _backend().paged_append(s.desc)
        return {"q": s.q_out, "k": s.k_pool, "v": s.v_pool}
    if s.op == "attention":
        _backend().paged_attention(s.desc)
        return s.out
    _backend().sample(s.desc)
    return {"ids": s.ids, "probs": s.probs}


# ---------------------------------------------------------------------------------------------- plain forms
def _plain_append(s):
    case, hd, rot = s.case, s.case["head_dim"], s.case["rope_dim"]
    h, h_kv = case["n_head"], case["n_head_kv"]
    row = torch.arange(s.n_rows, device="cuda")
    seq = torch.searchsorted(s.row_start, row, right=True) - 1
    pos = s.n_kv[seq] - s.row_start[seq + 1] + row
    pair = torch.arange(rot // 2, device="cuda", dtype=torch.float64)
    angle = (pos.double()[:, None] * torch.pow(torch.tensor(case["base"], dtype=torch.float64, device="cuda"), -2 * pair / rot))[:, None, :]
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    a = torch.arange(0, rot, 2, device="cuda") if case["mode"] == 0 else torch.arange(rot // 2, device="cuda")
    b = a + 1 if case["mode"] == 0 else a + rot // 2
    x = s.qkv.view(s.n_rows, h + 2 * h_kv, hd).float()
    turned = x[:, :h + h_kv].clone()
    turned[:, :, a] = x[:, :h + h_kv, a] * cos - x[:, :h + h_kv, b] * sin
    turned[:, :, b] = x[:, :h + h_kv, a] * sin + x[:, :h + h_kv, b] * cos
    k_pages, v_pages = _paged_views(s)
    page, slot = s.table[seq, pos // case["page"]].long(), (pos % case["page"]).long()
    k_pages[page, slot] = turned[:, h:].half()
    v_pages[page, slot] = x[:, h + h_kv:].half()
    s.q_out.copy_(turned[:, :h].half())
    return {"q": s.q_out, "k": s.k_pool, "v": s.v_pool}


def _plain_attention(s):
    case, hd, h, h_kv = s.case, s.case["head_dim"], s.case["n_head"], s.case["n_head_kv"]
    k_pages, v_pages = _paged_views(s)
    alike = {}
    for i, n in enumerate(s.rows):                          # sequences with the same number of new tokens go together, padded to the longest
        alike.setdefault(n, []).append(i)
    for n, seqs in alike.items():
        longest = max(s.kv[i] for i in seqs)
        which = torch.tensor(seqs, device="cuda")
        pos = torch.arange(longest, device="cuda")
        page, slot = s.table[which][:, pos // case["page"]].clamp(min=0).long(), pos % case["page"]
        k, v = (x[page, slot].permute(0, 2, 1, 3).float() for x in (k_pages, v_pages))          # [sequence][head][position][element]
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


def _plain_sample(s):
    """In 64 bits: which token a number falls on is decided next to the borders of the sums."""
    cold = (s.temperature == 0)[:, None]
    logits, order = torch.sort(s.logits, dim=1, descending=True, stable=True)
    z = logits.double() / torch.where(cold, 1.0, s.temperature[:, None].double())
    w = torch.exp(z - z[:, :1])
    rank = torch.arange(w.shape[1], device="cuda")
    top_k = torch.where(s.top_k > 0, s.top_k, w.shape[1])[:, None]
    w = torch.where(rank < torch.where(cold, 1, top_k), w, 0.0)
    before = torch.cumsum(w, 1) - w
    w = torch.where((s.top_p[:, None] >= 1) | (before < s.top_p[:, None].double() * w.sum(1, keepdim=True)), w, 0.0)
    w = torch.where(w >= s.min_p[:, None].double(), w, 0.0)
    w = torch.zeros_like(w).scatter_(1, order, w)
    upto = torch.cumsum(w, 1)
    total = upto[:, -1:]
    last = (w.shape[1] - 1 - torch.argmax((w > 0).flip(1).int(), 1))
    ids = torch.minimum((upto <= s.uniform[:, None].double() * total).sum(1), last)
    return {"ids": ids.int(), "probs": (w.gather(1, ids[:, None]) / total)[:, 0].float()}


def run(state):
    if own:
        return _own(state)
    return {"append": _plain_append, "attention": _plain_attention, "sample": _plain_sample}[state.op](state)


# ---------------------------------------------------------------------------------------------- by the definition, in 64 bits
def _exact_append(s):
    case, hd, rot, h, h_kv = s.case, s.case["head_dim"], s.case["rope_dim"], s.case["n_head"], s.case["n_head_kv"]
    pools = [s.k_pool.double(), s.v_pool.double()]
    views = pools if case["layout"] == "token" else [p.transpose(1, 2) for p in pools]
    q_out = torch.empty((s.n_rows, h, hd), dtype=torch.float64, device="cuda")
    speeds = torch.tensor([case["base"] ** (-2.0 * i / rot) for i in range(rot // 2)], dtype=torch.float64, device="cuda")
    first = 0
    for i, (n, kv) in enumerate(zip(s.rows, s.kv)):
        x = s.qkv[first:first + n].double().view(n, h + 2 * h_kv, hd)
        where = torch.arange(kv - n, kv, device="cuda")
        turn = torch.polar(torch.ones((n, rot // 2), dtype=torch.float64, device="cuda"), where.double()[:, None] * speeds)[:, None]
        head = x[:, :h + h_kv, :rot]
        pairs = head.reshape(n, -1, rot // 2, 2) if case["mode"] == 0 else torch.stack([head[..., :rot // 2], head[..., rot // 2:]], -1)
        turned = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
        turned = turned.reshape(n, -1, rot) if case["mode"] == 0 else torch.cat([turned[..., 0], turned[..., 1]], -1)
        full = torch.cat([turned, x[:, :h + h_kv, rot:]], -1)
        q_out[first:first + n] = full[:, :h]
        pages, slots = s.table[i][where // case["page"]].long(), where % case["page"]
        views[0][pages, slots] = full[:, h:]
        views[1][pages, slots] = x[:, h + h_kv:]
        first += n
    return {"q": q_out, "k": pools[0], "v": pools[1]}


def _exact_attention(s):
    case, hd, h, h_kv = s.case, s.case["head_dim"], s.case["n_head"], s.case["n_head_kv"]
    k_pages, v_pages = _paged_views(s)
    out = torch.empty((s.n_rows, h, hd), dtype=torch.float64, device="cuda")
    first = 0
    for i, (n, kv) in enumerate(zip(s.rows, s.kv)):
        pages = s.table[i, :-(-kv // case["page"])].long()
        k, v = (x[pages].flatten(0, 1)[:kv] for x in (k_pages, v_pages))                      # [position][head][element]
        block = max(1, int(2e8) // (kv * (h // h_kv)))
        for g in range(h_kv):
            kg, vg = k[:, g].double(), v[:, g].double()
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


def _exact_sample(s):
    logits = s.logits.cpu().numpy().astype(np.float64)
    setting = {k: getattr(s, k).cpu().numpy() for k in ("temperature", "top_k", "top_p", "min_p", "uniform")}
    ids, probs = np.empty(len(logits), dtype=np.int32), np.empty(len(logits))
    for r, x in enumerate(logits):
        t, k, p, least, u = (float(setting[n][r]) for n in ("temperature", "top_k", "top_p", "min_p", "uniform"))
        if t == 0:
            ids[r], probs[r] = int(np.argmax(x)), 1.0
            continue
        w = np.exp((x - x.max()) / t)
        kept = np.lexsort((np.arange(len(x)), -x))
        kept = kept[:int(k)] if k > 0 else kept
        if p < 1:
            sums = np.concatenate([[0.0], np.cumsum(w[kept])])
            kept = kept[sums[:-1] < p * sums[-1]]
        kept = np.sort(kept[w[kept] >= least])
        sums = np.cumsum(w[kept])
        at = min(int(np.searchsorted(sums, u * sums[-1], side="right")), len(kept) - 1)
        ids[r], probs[r] = kept[at], w[kept[at]] / sums[-1]
    return {"ids": torch.from_numpy(ids), "probs": torch.from_numpy(probs)}


def exact(case, seed):
    if case["op"] == "attention" and work(case)["flops"] > 8e13:
        return None
    s = prepare(case, seed)
    return {"append": _exact_append, "attention": _exact_attention, "sample": _exact_sample}[case["op"]](s)


# ---------------------------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    if case["op"] == "sample":
        return {"bytes": case["rows"] * (4 * case["vocab"] + 28), "flops": 2 * case["rows"] * case["vocab"]}
    rows, kv = _lengths(case)
    h, h_kv, hd, n = case["n_head"], case["n_head_kv"], case["head_dim"], sum(rows)
    if case["op"] == "append":
        size = 2 if case["dtype"] == "f16" else 4
        return {"bytes": n * (h + 2 * h_kv) * hd * (size + 2), "flops": 3 * n * (h + h_kv) * case["rope_dim"]}
    reach = case["window"] or 1 << 40
    read = sum(min(k, r + reach - 1) for r, k in zip(rows, kv))                # positions that some row of the sequence sees
    pairs = 0
    for r, k in zip(rows, kv):                                                 # row i sees min(k - r + i + 1, reach) positions
        full = max(0, min(r, reach - (k - r)))                                 # rows that see their whole past
        pairs += full * (k - r) + full * (full + 1) // 2 + (r - full) * reach if reach < 1 << 40 else r * (k - r) + r * (r + 1) // 2
    return {"bytes": 4 * n * h * hd + 4 * read * h_kv * hd, "flops": 4 * pairs * h * hd}
