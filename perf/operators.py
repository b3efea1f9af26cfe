"""What the operators around the INT8 KV cache cost: attention of drafted token trees, accumulated attention weight,
the choice of the cache rows to keep, and their compaction.

``listed()`` and ``draw()`` give cases, ``prepare()`` makes a case's inputs on the GPU, ``run()`` makes one pass (in
elementary torch operations, or through the library where ``own`` is true), ``exact()`` is the definition in 64 bits
and ``work()`` the bytes and operations that a pass cannot do without.

The head counts and head sizes are those of ``workloads.SPECS`` (8 / 8 heads of 64, 32 / 32, 32 / 8 and 64 / 8 heads
of 128), and so are the ranges of the cached lengths.
"""
from __future__ import annotations

import math
import random

import torch

own = False

GROUP = 8  # channels per scale


# ------------------------------------------------------------------------------------------------------------------
# cases
# ------------------------------------------------------------------------------------------------------------------

def _case(name, op, heads, kv_heads, dim, batch, lo, hi, shape, **more):
    c = dict(name=name, op=op, heads=heads, kv_heads=kv_heads, dim=dim, batch=batch, lo=lo, hi=hi, shape=shape,
             layout=0, page=0, layers=1)
    c.update(more)
    return c


def listed():
    return [
        # one speculative step of a small batch of short dialogues: latency counts
        _case("tree short", "tree", 8, 8, 64, 4, 17, 255, 1, n_lo=3, n_hi=7),
        # a serving batch, short trees of ragged sizes (some sequences verify a single token)
        _case("tree batch", "tree", 32, 8, 128, 32, 256, 8192, 2, n_lo=1, n_hi=16),
        # a large batch with bigger trees, 8 query heads share a kv head
        _case("tree wide", "tree", 64, 8, 128, 64, 64, 8192, 3, n_lo=25, n_hi=33),
        # few long contexts in a paged, head-major cache, large trees
        _case("tree long paged", "tree", 32, 8, 128, 4, 32768, 131072, 4, n_lo=57, n_hi=64, layout=3, page=128),
        # the weights that one decode step adds, small batch
        _case("weight short", "weight", 8, 8, 64, 4, 17, 255, 5, n_lo=1, n_hi=1, steps=20),
        # the weights that one decode step of a serving batch adds, one query head per kv head
        _case("weight decode", "weight", 32, 32, 128, 64, 128, 4096, 6, n_lo=1, n_hi=1, steps=200),
        # the observation window at the end of long prompts, before the first eviction
        _case("weight window", "weight", 32, 8, 128, 4, 8192, 32768, 7, n_lo=29, n_hi=32, steps=0),
        # which rows to keep, small batch
        _case("select short", "select", 8, 8, 64, 4, 17, 255, 8, keep=50, sink=4, recent=16),
        # which rows of long contexts to keep
        _case("select long", "select", 32, 8, 128, 16, 32768, 131072, 9, keep=4096, sink=4, recent=256),
        # the accepted paths of a batch of trees: a few rows of every layer of a sequence move to the front
        _case("compact path", "compact", 32, 8, 128, 32, 40, 130, 10, layers=32, n_lo=8, n_hi=16, path=6),
        # the survivors of an eviction: a kept list for every kv head, weights move along
        _case("compact evict", "compact", 32, 8, 128, 16, 4096, 16384, 11, keep=2048, sink=4, recent=256),
        # the same for few long contexts in a paged, head-major cache
        _case("compact paged", "compact", 32, 8, 128, 4, 32768, 131072, 12, keep=16001, sink=4, recent=1024, layout=3,
              page=128),
    ]


def _log_between(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("tree", "tree", "weight", "weight", "select", "compact"))
    heads, kv_heads, dim = rng.choice(((8, 8, 64), (32, 32, 128), (32, 8, 128), (64, 8, 128)))
    batch = _log_between(rng, 1, 64)
    # cached elements of the largest listed cases: some 4 * 64 Ki positions of 8 heads of 128
    most = min(131072, (1 << 27) // (batch * kv_heads * dim))
    hi = _log_between(rng, 64, max(64, most))
    lo = max(1, int(hi * rng.uniform(0.05, 1.0)))
    c = dict(op=op, heads=heads, kv_heads=kv_heads, dim=dim, batch=batch, lo=lo, hi=hi, shape=rng.randrange(1 << 30),
             layout=rng.choice((0, 3)), page=rng.choice((0, 0, 16, 48, 128)), layers=1)
    if op == "tree":
        c["n_hi"] = _log_between(rng, 1, 64)
        c["n_lo"] = rng.randint(1, c["n_hi"])
    elif op == "weight":
        c["n_hi"] = rng.choice((1, 1, _log_between(rng, 2, 32)))
        c["n_lo"] = rng.randint(1, c["n_hi"])
        c["steps"] = rng.choice((0, 10, 300))
    elif op == "select" or rng.random() < 0.7:
        c["keep"] = max(1, int(hi * rng.uniform(0.05, 0.6)))
        c["sink"] = rng.choice((0, 1, 4))
        c["recent"] = rng.choice((0, 16, 129))
    else:
        c["layers"] = rng.choice((1, 2, 7))
        c["hi"] = min(c["hi"], 2048)
        c["lo"] = min(c["lo"], c["hi"])
        c["n_hi"] = _log_between(rng, 2, 64)
        c["n_lo"] = rng.randint(1, c["n_hi"])
        c["path"] = rng.randint(1, 9)
    return c


def _shape(case):
    """Lengths, drafts, parents, rows: what a case fixes whatever its seed (lists of ints)."""
    rng = random.Random(case["shape"])
    hist = [rng.randint(case["lo"], case["hi"]) for _ in range(case["batch"])]
    hist[0] = case["hi"]
    n = [rng.randint(case["n_lo"], case["n_hi"]) if "n_lo" in case else 0 for _ in hist]
    if "n_hi" in case:
        n[-1] = case["n_hi"]
    # a drafted token hangs under one of the last few before it, or under the history
    parents = [[-1 if i == 0 else rng.randint(max(-1, i - 6), i - 1) for i in range(m)] for m in n]
    # decode and window queries are the last tokens of their sequence
    start = [max(0, h - m) for h, m in zip(hist, n)] if case["op"] == "weight" else hist
    total = [s + m for s, m in zip(start, n)]
    gaps = [rng.randint(0, 9) for _ in hist]  # rows of others between two sequences
    page = case["page"]
    if page:
        pages = [-(-t // page) for t in total]
        order = list(range(sum(pages)))
        rng.shuffle(order)
        starts, at = [], 0
        for p in pages:
            starts.append([r * page for r in order[at:at + p]] + [0] * (max(pages) - p))
            at += p
        rows = sum(pages) * page
    else:
        starts, rows = [], 0
        for t, g in zip(total, gaps):
            starts.append(rows)
            rows += t + g
    return dict(start=start, n=n, total=total, parents=parents, starts=starts, rows=rows, max_n=max(n),
                max_total=max(total))


def _depths(parents):
    out = []
    for p in parents:
        out.append(1 if p < 0 else out[p] + 1)
    return out


def work(case):
    s = _shape(case)
    h, g, d = case["heads"], case["kv_heads"], case["dim"]
    row = d + d // GROUP * 2  # codes and scales of one row of one head, K or V
    tokens, total = sum(s["n"]), sum(s["total"])
    index = 8 * (4 * case["batch"] + 1) + (8 * len(s["starts"][0]) * case["batch"] if case["page"] else 0)
    if case["op"] == "tree":
        pairs = sum(n * a + sum(_depths(p)) for n, a, p in zip(s["n"], s["start"], s["parents"]))
        return dict(bytes=total * g * 2 * row + tokens * (h * d * 4 + 8) + index, flops=4 * d * h * pairs)
    if case["op"] == "weight":
        pairs = sum(n * a + n * (n + 1) // 2 for n, a in zip(s["n"], s["start"]))
        return dict(bytes=total * g * (row + 8) + tokens * h * d * 2 + index, flops=2 * d * h * pairs)
    if case["op"] == "select":
        return dict(bytes=g * (4 * total + 8 * case["batch"] * case["keep"]) + index, flops=g * total)
    if "path" in case:
        moved = sum(max(0, min(case["path"], n) - 1) for n in s["n"])  # the first of a path stays where it is
        return dict(bytes=moved * case["layers"] * g * 2 * row * 2 + 8 * case["batch"] * case["path"] + index, flops=0)
    moved = sum(max(0, min(case["keep"], t) - case["sink"]) if t > case["keep"] else 0 for t in s["total"])
    cleared = sum(max(0, t - case["keep"]) for t in s["total"])
    return dict(bytes=moved * g * (4 * row + 8) + 4 * g * cleared + 8 * g * case["batch"] * case["keep"] + index, flops=0)


# ------------------------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------------------------

def _shapes(case, rows):
    h, d, layers = case["kv_heads"], case["dim"], case["layers"]
    lead = (rows, layers, 2, h) if case["layout"] == 0 else (layers, 2, h, rows)
    return lead + (d,), lead + (d // GROUP,)


def _fill(case, rows, gen):
    """A cache of normal K and V, every 16th K channel eight times as large (outlier channels), quantised in groups."""
    code_shape, scale_shape = _shapes(case, rows)
    x = torch.randn(code_shape, generator=gen, device="cuda")
    k = x[:, :, 0] if case["layout"] == 0 else x[:, 0]
    k[..., ::16] *= 8
    x = x.view(scale_shape + (GROUP,))
    scale = (x.abs().amax(-1) / 127).half()
    x /= scale.float().clamp_min(1e-8).unsqueeze(-1)
    return x.round_().clamp_(-127, 127).to(torch.int8).view(code_shape), scale


def prepare(case, seed):
    s = _shape(case)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    ints = lambda v: torch.tensor(v, dtype=torch.int64, device="cuda")  # noqa: E731
    d = dict(case=dict(case), cachestarts=ints(s["starts"]), start_pos=ints(s["start"]), kvlens=ints(s["total"]),
             max_n=s["max_n"], max_total=s["max_total"])
    batch, g = case["batch"], case["kv_heads"]
    if case["op"] in ("tree", "weight"):
        tokens = sum(s["n"])
        d["seqstarts"] = ints([0] + s["n"]).cumsum(0)
        d["query"] = torch.randn((tokens, case["heads"], case["dim"]), generator=gen, device="cuda").half()
        if case["op"] == "tree":
            d["parents"] = ints([p for ps in s["parents"] for p in ps])
    if case["op"] != "select":
        d["cache"], d["scale"] = _fill(case, s["rows"], gen)
    if case["op"] in ("weight", "select") or "keep" in case:
        # what earlier steps left: heavy-tailed sums, spread over the sequence; `steps` of them, or 100
        w = torch.rand((case["layers"], g, s["rows"]), generator=gen, device="cuda").clamp_min(1e-6)
        d["weight"] = w.pow(-0.7) * (case.get("steps", 100) / s["max_total"])
    if case["op"] == "select":
        d["budgets"] = ints([case["keep"]] * batch)
    if case["op"] == "compact":
        if "path" in case:  # ascending drafts of each sequence, the first one among them
            score = torch.rand((batch, 1, s["max_n"]), generator=gen, device="cuda")
            here = torch.arange(s["max_n"], device="cuda")
            score[..., 0] = 2
            score = torch.where(here < ints(s["n"])[:, None, None], score, -1.0)
            d["kept"] = _ascending(score, ints([case["path"]] * batch), case["path"])
            d["base"] = d["start_pos"]
        else:
            score = torch.rand((batch, g, s["max_total"]), generator=gen, device="cuda")
            here = torch.arange(s["max_total"], device="cuda")
            n = d["kvlens"][:, None, None]
            score = torch.where((here < case["sink"]) | (here >= n - case["recent"]), 2.0, score)
            score = torch.where(here < n, score, -1.0)
            d["kept"] = _ascending(score, ints([case["keep"]] * batch), case["keep"])
            d["base"] = torch.zeros_like(d["kvlens"])
    return d


def _ascending(score, budgets, width):
    """The positions of the `budgets` highest scores >= 0 of each row, lowest first among equals, in ascending order;
    -1 behind them.  [B, H, P] -> [B, H, width]."""
    order = score.sort(dim=-1, descending=True, stable=True).indices[..., :width]
    rank = torch.arange(order.shape[-1], device=score.device)
    use = (rank < budgets[:, None, None]) & (score.gather(-1, order) >= 0)
    big = score.shape[-1]
    order = torch.where(use, order, big).sort(dim=-1).values
    order = torch.where(order == big, -1, order)
    return torch.nn.functional.pad(order, (0, width - order.shape[-1]), value=-1)


# ------------------------------------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------------------------------------

def run(state):
    op = state["case"]["op"]
    if own:
        return _own_run(op, state)
    if op == "tree":
        return _plain_tree(state)
    if op == "weight":
        return _plain_weight(state)
    if op == "select":
        return _plain_select(state)
    return _plain_compact(state)


def _own_op(op, case):
    import __graft_entry__
    __graft_entry__.load_package()
    from ppl_nn_b200 import ops
    cache = dict(num_layer=case["layers"], layer_idx=0, quant_bit=8, cache_mode=1 if case["page"] else 0,
                 cache_layout=case["layout"], page_size=case["page"] or 128)
    heads = dict(num_heads=case["heads"], num_kv_heads=case["kv_heads"], head_dim=case["dim"])
    if op == "tree":
        return ops.TreeAttention(ops.MultiHeadCacheAttentionParam(**heads, **cache))
    if op == "weight":
        return ops.AttentionWeight(ops.MultiHeadCacheAttentionParam(**heads, **cache))
    if op == "select":
        return ops.KeyValueCacheEvict(ops.KeyValueCacheEvictParam(**cache, sink=case["sink"], recent=case["recent"]))
    return ops.KeyValueCacheCompact(ops.KeyValueCacheParam(**cache))


def _own_run(op, s):
    if "op" not in s:  # a program makes its operators once
        s["op"] = _own_op(op, s["case"])
    f = s["op"].forward
    if op == "tree":
        return f(s["query"], s["parents"], s["seqstarts"], s["cachestarts"], s["start_pos"], s["max_n"], s["max_total"],
                 s["cache"], s["scale"])
    if op == "weight":
        return f(s["query"], s["seqstarts"], s["cachestarts"], s["start_pos"], s["max_n"], s["max_total"], s["cache"],
                 s["scale"], s["weight"])
    if op == "select":
        return f(s["weight"], s["cachestarts"], s["kvlens"], s["budgets"], s["max_total"], s["case"]["keep"])
    f(s["kept"], s["cachestarts"], s["base"], s["kvlens"], s["max_total"], s["cache"], s["scale"],
      weight=s.get("weight"), num_layers=s["case"]["layers"])
    return [s[k] for k in ("cache", "scale", "weight") if k in s]


def _rows(s, pos):
    """Cache rows of the positions [B, P] (positions beyond a sequence's end are read as its last)."""
    pos = torch.minimum(pos, s["kvlens"][:, None] - 1).clamp_min(0)
    page = s["case"]["page"]
    if page:
        return s["cachestarts"].gather(1, pos // page) + pos % page
    return s["cachestarts"][:, None] + pos


def _dense(s, which, rows):
    """K (0) or V (1) of the rows [B, P] as [B, Hkv, P, D] in fp32."""
    pick = (lambda t: t[rows, 0, which].transpose(1, 2)) if s["case"]["layout"] == 0 else (
        lambda t: t[0, which][:, rows].transpose(0, 1))
    codes, scale = pick(s["cache"]), pick(s["scale"])
    x = codes.float().unflatten(-1, (-1, GROUP)) * scale.float().unsqueeze(-1)
    return x.flatten(-2)


def _padded_queries(s):
    """[B, Hkv, N * group, D] in fp32, and for every slot of N whether it holds a token."""
    first, here = s["seqstarts"][:-1, None], torch.arange(s["max_n"], device="cuda")
    there = first + here < s["seqstarts"][1:, None]
    tok = torch.where(there, first + here, 0)
    q = s["query"].float()[tok]  # [B, N, H, D]
    g = s["case"]["kv_heads"]
    b, n, h, d = q.shape
    return q.view(b, n, g, h // g, d).transpose(1, 2).reshape(b, g, n * (h // g), d), there


def _softmax(scores, visible):
    """Softmax over the last axis of the visible places; rows that see nothing give zeros."""
    scores = torch.where(visible, scores, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    return p / p.sum(-1, keepdim=True).clamp_min(1e-30)


def _plain_tree(s):
    c = s["case"]
    pos = torch.arange(s["max_total"], device="cuda").expand(c["batch"], -1)
    rows = _rows(s, pos)
    q, there = _padded_queries(s)
    n, group = s["max_n"], c["heads"] // c["kv_heads"]
    # (I - P)^-1 = I + P + P^2 + ..: 1 where one drafted token is another or among its ancestors
    first = s["seqstarts"][:-1, None] + torch.arange(n, device="cuda")
    par = torch.where(there, s["parents"][torch.where(there, first, 0)], -1)
    eye = torch.eye(n, device="cuda")
    up = (par[..., None] == torch.arange(n, device="cuda")).float()
    anc = torch.linalg.solve_triangular(eye - up, eye.expand_as(up), upper=False, unitriangular=True) > 0.5
    start = s["start_pos"][:, None]
    off = (pos - start).clamp(0, n - 1)[:, None, :].expand(-1, n, -1)
    seen = ((pos < start)[:, None, :] | anc.gather(2, off)) & (pos < s["kvlens"][:, None])[:, None, :]
    seen = (seen & there[..., None]).repeat_interleave(group, 1)[:, None]
    p = _softmax(q @ _dense(s, 0, rows).transpose(2, 3) / math.sqrt(c["dim"]), seen)
    o = p @ _dense(s, 1, rows)  # [B, Hkv, N * group, D]
    o = o.view(c["batch"], c["kv_heads"], n, group, c["dim"]).transpose(1, 2).reshape(c["batch"], n, c["heads"], c["dim"])
    t = torch.arange(s["query"].shape[0], device="cuda")
    b = torch.searchsorted(s["seqstarts"], t, right=True) - 1
    return o[b, t - s["seqstarts"][b]].half()


def _plain_weight(s):
    c = s["case"]
    pos = torch.arange(s["max_total"], device="cuda").expand(c["batch"], -1)
    rows = _rows(s, pos)
    q, there = _padded_queries(s)
    last = s["start_pos"][:, None] + torch.arange(s["max_n"], device="cuda")
    seen = (pos[:, None, :] <= last[..., None]) & there[..., None]
    seen = seen.repeat_interleave(c["heads"] // c["kv_heads"], 1)[:, None]
    p = _softmax(q @ _dense(s, 0, rows).transpose(2, 3) / math.sqrt(c["dim"]), seen)
    w = p.sum(2)  # [B, Hkv, P]
    w = torch.where((pos < s["kvlens"][:, None])[:, None], w, 0.0)
    s["weight"][0].index_add_(1, rows.reshape(-1), w.transpose(0, 1).reshape(c["kv_heads"], -1))
    return s["weight"]


def _plain_select(s):
    c = s["case"]
    pos = torch.arange(s["max_total"], device="cuda").expand(c["batch"], -1)
    n = s["kvlens"][:, None, None]
    keep = torch.minimum(s["budgets"][:, None, None], n)
    recent = keep.clamp_max(c["recent"])
    sink = (keep - recent).clamp_max(c["sink"])
    w = s["weight"][0][:, _rows(s, pos)].transpose(0, 1)  # [B, Hkv, P], not negative
    pos = pos[:, None]
    w = torch.where((pos < sink) | (pos >= n - recent), math.inf, w)
    w = torch.where(pos < n, w, -1.0)
    return _ascending(w, s["budgets"], c["keep"])


def _plain_compact(s):
    c, kept = s["case"], s["kept"]
    batch, g, width = c["batch"], c["kv_heads"], kept.shape[-1]
    kept = kept.expand(batch, g, width)
    use = kept >= 0
    base = s["base"][:, None]
    src = _rows(s, (base + kept.clamp_min(0).reshape(batch, -1))).view(batch, g, width)[use]
    dst = _rows(s, (base + torch.arange(width, device="cuda").expand(batch, g, width).reshape(batch, -1)))
    dst = dst.view(batch, g, width)[use]
    head = torch.arange(g, device="cuda")[None, :, None].expand(batch, g, width)[use]
    if c["layout"] == 0:
        s["cache"][dst, :, :, head] = s["cache"][src, :, :, head]
        s["scale"][dst, :, :, head] = s["scale"][src, :, :, head]
    else:
        s["cache"][:, :, head, dst] = s["cache"][:, :, head, src]
        s["scale"][:, :, head, dst] = s["scale"][:, :, head, src]
    if "weight" not in s:
        return [s["cache"], s["scale"]]
    s["weight"][:, head, dst] = s["weight"][:, head, src]
    pos = torch.arange(s["max_total"], device="cuda").expand(batch, g, -1)
    behind = (pos >= s["base"][:, None, None] + use.sum(-1, keepdim=True)) & (pos < s["kvlens"][:, None, None])
    rows = _rows(s, pos[:, 0])[:, None].expand_as(pos)[behind]
    head = torch.arange(g, device="cuda")[None, :, None].expand_as(pos)[behind]
    s["weight"][:, head, rows] = 0.0
    return [s["cache"], s["scale"], s["weight"]]


# ------------------------------------------------------------------------------------------------------------------
# the definition in 64 bits, one sequence at a time
# ------------------------------------------------------------------------------------------------------------------

def _row_list(case, shape, b, positions):
    starts, page = shape["starts"][b], case["page"]
    if not page:
        return [starts + p for p in positions]
    return [starts[p // page] + p % page for p in positions]


def _values(case, state, which, rows, head):
    codes, scale = state["cache"], state["scale"]
    if case["layout"] == 0:
        codes, scale = codes[rows, 0, which, head], scale[rows, 0, which, head]
    else:
        codes, scale = codes[0, which, head, rows], scale[0, which, head, rows]
    return codes.double() * scale.double().repeat_interleave(GROUP, -1)


def exact(case, seed):
    shape, s = _shape(case), prepare(case, seed)
    if case["op"] == "select":
        return None  # positions, no computed numbers
    if case["op"] == "compact":
        return _exact_compact(case, shape, s)
    group, d = case["heads"] // case["kv_heads"], case["dim"]
    out = torch.zeros(s["query"].shape, dtype=torch.float64, device="cuda")
    weight = s["weight"].double() if case["op"] == "weight" else None
    first = 0
    for b, (start, n, total) in enumerate(zip(shape["start"], shape["n"], shape["total"])):
        rows = torch.tensor(_row_list(case, shape, b, range(total)), device="cuda")
        seen = torch.zeros((n, total), dtype=torch.bool)
        for i in range(n):
            if case["op"] == "weight":
                seen[i, :start + i + 1] = True
            else:
                seen[i, :start] = True
                a = i
                while a >= 0:
                    seen[i, start + a] = True
                    a = shape["parents"][b][a]
        hidden = ~seen.cuda()
        for g in range(case["kv_heads"]):
            q = s["query"][first:first + n, g * group:(g + 1) * group].double()
            k = _values(case, s, 0, rows, g)
            x = torch.einsum("nhd,pd->hnp", q, k) * d ** -0.5
            p = x.masked_fill(hidden, -math.inf).softmax(-1)
            if case["op"] == "weight":
                weight[0, g, rows] += p.sum((0, 1))
            else:
                out[first:first + n, g * group:(g + 1) * group] = torch.einsum("hnp,pd->nhd", p, _values(case, s, 1, rows, g))
        first += n
    return weight if case["op"] == "weight" else out


def _exact_compact(case, shape, s):
    old_scale, old_weight = s["scale"].double(), s["weight"].double() if "weight" in s else None
    scale, weight = old_scale.clone(), old_weight.clone() if "weight" in s else None
    kept = s["kept"].tolist()
    for b, total in enumerate(shape["total"]):
        base = shape["start"][b] if "path" in case else 0
        for g in range(case["kv_heads"]):
            mine = [k for k in kept[b][g if len(kept[b]) > 1 else 0] if k >= 0]
            src = torch.tensor(_row_list(case, shape, b, [base + k for k in mine]), device="cuda")
            dst = torch.tensor(_row_list(case, shape, b, range(base, base + len(mine))), device="cuda")
            if case["layout"] == 0:
                scale[dst, :, :, g] = old_scale[src, :, :, g]
            else:
                scale[:, :, g, dst] = old_scale[:, :, g, src]
            if weight is not None:
                weight[:, g, dst] = old_weight[:, g, src]
                weight[:, g, _row_list(case, shape, b, range(base + len(mine), total))] = 0
    return [None, scale, weight] if weight is not None else [None, scale]
