"""The operators around the INT8 cache as they are used together -- drafting, eviction, captured steps, several streams,
long caches -- and the forms of each that its own tests leave out."""
import numpy as np
import pytest

from test_cache_ops import HostCache, _params, _weight_call, dev, gpu, starts_of, weight_reference  # noqa: F401  (gpu is a fixture)
from test_tree_attention import draw_parents, run_tree, tree_reference

I64 = np.int64


def attention_param(hc, heads, layer=0, **kw):
    from ppl_nn_b200 import ops
    return ops.MultiHeadCacheAttentionParam(num_heads=heads, num_kv_heads=hc.heads, head_dim=hc.dim, **hc.param(layer), **kw)


def i64(x):
    return dev(np.array(x, dtype=I64))


# ---- refusals by the Python layer -----------------------------------------------------------------

def test_host_tensors_are_refused(pkg, built_lib):
    import torch
    from ppl_nn_b200 import ops
    hc = HostCache(np.random.default_rng(0), [5, 9], 2, 64)
    t = torch.from_numpy
    cache, scale, weight = t(hc.cache), t(hc.scale), t(hc.weight)
    q, one = torch.zeros(2, 4, 64, dtype=torch.float16), torch.zeros(2, dtype=torch.int64)
    seq = torch.tensor([0, 1, 2])
    p = attention_param(hc, 4)
    for call in (lambda: ops.TreeAttention(p).forward(q, None, seq, one, one, 1, 9, cache, scale),
                 lambda: ops.AttentionWeight(p).forward(q, seq, one, one, 1, 9, cache, scale, weight),
                 lambda: ops.KeyValueCacheEvict(ops.KeyValueCacheEvictParam(**hc.param())).forward(weight, one, one, one, 9, 4),
                 lambda: ops.KeyValueCacheCompact(ops.KeyValueCacheParam(**hc.param())).forward(
                     torch.zeros(2, 2, 4, dtype=torch.int64), one, one, one, 9, cache, scale)):
        with pytest.raises(ops.OpError):
            call()


def test_sizes_that_would_wrap_around_are_refused(pkg, built_lib):
    from ppl_nn_b200 import capi
    most = dict(num_heads=65535, num_kv_heads=65535, batch=65535, max_tokens=0x7fffffff, total_tokens=0x7fffffff)
    p = _params(built_lib, capi, **most, max_kvlen=1 << 27, max_seqlen=1)
    assert built_lib.status_str(built_lib.attn_weight_workspace_size(p)[0]) == "RC_UNSUPPORTED"
    assert built_lib.status_str(built_lib.kv_compact_workspace_size(p, 65535, 1 << 30, 1)[0]) == "RC_UNSUPPORTED"
    for longest in (1 << 31, 1 << 62):  # times the group of four: 2^64
        p = _params(built_lib, capi, max_seqlen=longest)
        assert built_lib.status_str(built_lib.attn_weight_workspace_size(p)[0]) == "RC_UNSUPPORTED"
        assert built_lib.status_str(_weight_call(built_lib, p)) == "RC_UNSUPPORTED"
    # the tree's work is cut into as many parts as there are places, however much it is
    p = _params(built_lib, capi, **most, max_kvlen=0x7fff0000, max_seqlen=1024)
    rc, n = built_lib.tree_attn_workspace_size(p)
    assert rc == capi.SUCCESS and n > 0x7fffffff * 16 * 8


@pytest.mark.parametrize("layout", [0, 3])
def test_a_cache_without_both_k_and_v_is_refused(pkg, built_lib, layout):
    """The rows' addresses follow from the attributes: a cache of K alone would be read beyond its end."""
    from ppl_nn_b200 import ops
    op = ops.KeyValueCacheCompact(ops.KeyValueCacheParam(num_layer=3, layer_idx=0, quant_bit=8, cache_layout=layout))

    def shapes(rows, layers, kv, heads, dim):
        lead = (rows, layers, kv, heads) if layout == 0 else (layers, kv, heads, rows)
        return lead + (dim,), lead + (dim // 8,)

    assert op._cache_shape(*shapes(50, 3, 2, 4, 64)) == (4, 64, 50)
    for bad in ((50, 3, 1, 4, 64), (50, 3, 3, 4, 64), (50, 2, 2, 4, 64), (50, 3, 0, 4, 64)):
        with pytest.raises(ops.OpError):
            op._cache_shape(*shapes(*bad))
    cache, scale = shapes(50, 3, 2, 4, 64)
    with pytest.raises(ops.OpError):
        op._cache_shape(cache, scale[:-1] + (4,))


@pytest.mark.gpu
def test_calls_without_work_leave_no_status(gpu, pkg):  # noqa: F811
    import torch
    from ppl_nn_b200 import ops
    hc = HostCache(np.random.default_rng(0), [5, 9], 2, 64)
    cache, scale, weight, none = dev(hc.cache), dev(hc.scale), dev(hc.weight), i64([])
    q = torch.zeros(0, 4, 64, dtype=torch.float16, device=gpu)
    p = attention_param(hc, 4)
    tree, weigh = ops.TreeAttention(p), ops.AttentionWeight(p)
    evict = ops.KeyValueCacheEvict(ops.KeyValueCacheEvictParam(**hc.param()))
    compact = ops.KeyValueCacheCompact(ops.KeyValueCacheParam(**hc.param()))
    junk = torch.full((1 << 16,), 255, dtype=torch.uint8, device=gpu)  # what a new workspace would hold
    del junk
    tree.forward(q, None, i64([0]), none, none, 0, 0, cache, scale)
    weigh.forward(q, i64([0]), none, none, 0, 0, cache, scale, weight)
    tree.forward(q, None, i64([0, 0, 0]), dev(hc.starts), i64([5, 9]), 0, 9, cache, scale)
    assert evict.forward(weight, none, none, none, 0, 4).shape == (0, 2, 4)
    assert evict.forward(weight, dev(hc.starts), i64([5, 9]), i64([0, 0]), 9, 0).shape == (2, 2, 0)
    compact.forward(i64(np.zeros((2, 1, 0))), dev(hc.starts), i64([0, 0]), i64([5, 9]), 9, cache, scale)
    assert [o.device_status() for o in (tree, weigh, evict, compact)] == [0] * 4
    assert np.array_equal(weight.cpu().numpy(), hc.weight) and np.array_equal(cache.cpu().numpy(), hc.cache)
    with pytest.raises(ops.OpError):
        ops.KeyValueCacheCompact(ops.KeyValueCacheParam(**hc.param(), num_repeat=2)).forward(
            i64(np.zeros((2, 1, 1))), dev(hc.starts), i64([0, 0]), i64([5, 9]), 9, cache, scale)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [[2, 3], [40, 9]])  # kept scores, and scores formed twice
def test_sequences_that_are_left_out_are_reported(gpu, pkg, n):  # noqa: F811
    """Rows that are not the query's, starts below zero and bounds that leave nothing: what cannot be served is reported,
    the others are served."""
    from ppl_nn_b200 import capi, ops
    rng = np.random.default_rng(n[0])
    start = [60, 200]
    hc = HostCache(rng, [s + m for s, m in zip(start, n)], 2, 64)
    q = rng.standard_normal((sum(n), 8, 64)).astype(np.float16)
    parents = sum([draw_parents(rng, m, "tree") for m in n], [])
    tree, weigh = ops.TreeAttention(attention_param(hc, 8)), ops.AttentionWeight(attention_param(hc, 8))
    lone = HostCache(rng, [hc.lens[0]], 2, 64)  # the first sequence by itself
    lone.starts, lone.cache, lone.scale, lone.weight, lone.max_tokens = hc.starts[:1], hc.cache, hc.scale, hc.weight, hc.max_tokens
    want, tol = weight_reference(lone, q, start[:1], n[:1], 8, 0, True)
    for seq, first in (([0, n[0], sum(n) + 1], start), ([0, n[0], n[0] - 1], start), ([0, n[0], sum(n)], [60, -1]),
                       ([0, n[0], sum(n)], [60, -(1 << 62)])):
        weight = dev(hc.weight)
        weigh.forward(dev(q), i64(seq), dev(hc.starts), i64(first), max(n), hc.max_len, dev(hc.cache), dev(hc.scale), weight)
        assert weigh.device_status() == capi.DEV_LENGTH_CLAMPED, (seq, first)
        assert np.all(np.abs(weight.cpu().numpy() - want) <= tol)
        tree.forward(dev(q), i64(parents), i64(seq), dev(hc.starts), i64(first), max(n), hc.max_len, dev(hc.cache), dev(hc.scale))
        assert tree.device_status() == capi.DEV_LENGTH_CLAMPED, (seq, first)
    for most_n, most_len in ((0, hc.max_len), (max(n), 0), (0, 0)):
        weight = dev(hc.weight)
        weigh.forward(dev(q), dev(starts_of(n)), dev(hc.starts), i64(start), most_n, most_len, dev(hc.cache), dev(hc.scale), weight)
        assert weigh.device_status() == capi.DEV_LENGTH_CLAMPED
        assert np.array_equal(weight.cpu().numpy(), hc.weight)
        tree.forward(dev(q), i64(parents), dev(starts_of(n)), dev(hc.starts), i64(start), most_n, most_len, dev(hc.cache), dev(hc.scale))
        assert tree.device_status() == capi.DEV_LENGTH_CLAMPED
    # a sequence without tokens, wherever it starts: nothing is left out
    for seq in ([0, n[0], n[0]], [0, 0, n[1]]):
        for far in (-1, 1 << 40):
            first = [far if seq[b] == seq[b + 1] else start[b] for b in range(2)]
            weight = dev(hc.weight)
            weigh.forward(dev(q), i64(seq), dev(hc.starts), i64(first), max(n), hc.max_len, dev(hc.cache), dev(hc.scale), weight)
            tree.forward(dev(q), i64(parents), i64(seq), dev(hc.starts), i64(first), max(n), hc.max_len, dev(hc.cache), dev(hc.scale))
            assert weigh.device_status() == 0, (seq, far)
            # (the second sequence's tokens are the first ones here: their parents are other's, and reported)
            assert tree.device_status() in ((0,) if seq[1] else (0, capi.DEV_PARENT_INVALID)), (seq, far)
            if seq[1]:
                assert np.all(np.abs(weight.cpu().numpy() - want) <= tol)
    # only padding: nothing is left out
    weigh.forward(dev(q), i64([0, 0, 0]), dev(hc.starts), i64(start), 0, hc.max_len, dev(hc.cache), dev(hc.scale), weight)
    tree.forward(dev(q), i64(parents), i64([0, 0, 0]), dev(hc.starts), i64(start), 0, hc.max_len, dev(hc.cache), dev(hc.scale))
    assert weigh.device_status() == 0 and tree.device_status() == 0


def test_kept_scores_take_a_bounded_workspace(pkg, built_lib):
    """64 sequences whose bound is 131072 positions, whatever their lengths: 8.6 GB of scores, which are formed twice."""
    from ppl_nn_b200 import capi
    bounds = dict(num_heads=64, num_kv_heads=8, batch=64, total_tokens=256, max_tokens=1 << 20)
    size = lambda **kw: built_lib.attn_weight_workspace_size(_params(built_lib, capi, **bounds, **kw))  # noqa: E731
    for max_seqlen in (1, 2, 4):
        for max_kvlen in (1 << 14, 1 << 17, 1 << 19, 1 << 22):
            rc, n = size(max_seqlen=max_seqlen, max_kvlen=max_kvlen)
            parts = 8 * 256 * 64 * (max_kvlen // 512 + 2)  # maxima and sums of the rows' chunks
            assert rc == capi.SUCCESS and n <= (4 << 30) + parts
    assert size(max_seqlen=4, max_kvlen=1 << 16)[1] > 4 << 30  # up to the limit they are kept


@pytest.mark.gpu
@pytest.mark.parametrize("heads,n,bound", [(2, [1, 1, 1], 140000000), (8, [4, 1, 3], 12000000)])
def test_weights_under_roomy_bounds(gpu, pkg, heads, n, bound):  # noqa: F811
    """Short sequences under a bound that would ask for more CTAs than a grid dimension has, or (32 rows) for more kept
    scores than there is room for."""
    from ppl_nn_b200 import ops
    rng = np.random.default_rng(heads)
    start = [700, 0, 64]
    hc = HostCache(rng, [s + m for s, m in zip(start, n)], 1 if heads == 8 else 2, 64)
    q = rng.standard_normal((sum(n), heads, 64)).astype(np.float16)
    want, tol = weight_reference(hc, q, start, n, heads, 0, True)
    op = ops.AttentionWeight(attention_param(hc, heads))
    weight = dev(hc.weight)
    op.forward(dev(q), dev(starts_of(n)), dev(hc.starts), i64(start), max(n), bound, dev(hc.cache), dev(hc.scale), weight)
    assert op.device_status() == 0
    assert np.all(np.abs(weight.cpu().numpy() - want) <= tol)


@pytest.mark.gpu
def test_wrong_types_and_shapes_are_refused(gpu, pkg):  # noqa: F811
    import torch
    from ppl_nn_b200 import ops
    hc = HostCache(np.random.default_rng(0), [5, 9], 2, 64)
    good = dict(q=torch.zeros(2, 4, 64, dtype=torch.float16, device=gpu), parents=i64([-1, -1]), seq=i64([0, 1, 2]),
                cs=dev(hc.starts), start=i64([4, 8]), cache=dev(hc.cache), scale=dev(hc.scale), weight=dev(hc.weight),
                kept=i64(np.zeros((2, 2, 3))), base=i64([0, 0]), lens=i64([5, 9]), budgets=i64([3, 3]))
    p = attention_param(hc, 4)
    tree, weigh = ops.TreeAttention(p), ops.AttentionWeight(p)
    evict = ops.KeyValueCacheEvict(ops.KeyValueCacheEvictParam(**hc.param()))
    compact = ops.KeyValueCacheCompact(ops.KeyValueCacheParam(**hc.param()))

    def calls(d):
        return dict(
            tree=lambda: tree.forward(d["q"], d["parents"], d["seq"], d["cs"], d["start"], 1, 9, d["cache"], d["scale"]),
            weight=lambda: weigh.forward(d["q"], d["seq"], d["cs"], d["start"], 1, 9, d["cache"], d["scale"], d["weight"]),
            evict=lambda: evict.forward(d["weight"], d["cs"], d["lens"], d["budgets"], 9, 3),
            compact=lambda: compact.forward(d["kept"], d["cs"], d["base"], d["lens"], 9, d["cache"], d["scale"], d["weight"]))

    for f in calls(good).values():  # the calls themselves are right (kept: position 0 alone, then not ascending)
        f()
    torch.cuda.synchronize()
    for name, bad, which in (
            ("q", good["q"].float(), "tree weight"), ("q", good["q"][:, :3], "tree weight"),
            ("q", good["q"].transpose(0, 1).contiguous().transpose(0, 1), "tree weight"),
            ("parents", good["parents"].int(), "tree"), ("parents", i64([-1]), "tree"),
            ("seq", i64([0, 1]), "tree weight"), ("seq", good["seq"].int(), "tree weight"),
            ("seq", i64([[0], [1], [2]]), "tree weight"), ("start", i64([[4], [8]]), "tree weight"),
            ("cs", good["cs"][:1], "tree weight evict compact"), ("cs", good["cs"].cpu(), "tree weight evict compact"),
            ("cs", good["cs"][:, None].contiguous(), "tree weight evict compact"),
            ("cache", good["cache"].half(), "tree weight compact"), ("cache", good["cache"][..., :32].contiguous(), "tree weight compact"),
            ("scale", good["scale"].float(), "tree weight compact"), ("scale", None, "tree weight compact"),
            ("scale", good["scale"][:3], "tree weight compact"),
            ("weight", good["weight"].double(), "weight evict compact"), ("weight", good["weight"][0], "weight evict compact"),
            ("weight", good["weight"][..., 1:].contiguous(), "weight compact"),
            ("lens", i64([[5], [9]]), "evict compact"), ("budgets", i64([3]), "evict"),
            ("base", i64([0]), "compact"), ("kept", i64(np.zeros((2, 3, 3))), "compact"), ("kept", i64(np.zeros((2, 3))), "compact"),
            ("kept", good["kept"].int(), "compact")):
        for op in which.split():
            with pytest.raises(ops.OpError):
                calls(dict(good, **{name: bad}))[op]()
    with pytest.raises(ops.OpError):  # other parts of the call still read the query
        tree.forward(good["q"], None, good["seq"], good["cs"], good["start"], 1, 9, good["cache"], good["scale"],
                     attn_output=good["q"])
    if torch.cuda.device_count() > 1:
        with pytest.raises(ops.OpError):
            calls(dict(good, cs=good["cs"].to("cuda:1")))["tree"]()


# ---- a run of them, as they are used -----------------------------------------------------------------

def decode_output(hc, cache, scale, starts, heads, start, q, k, v):
    """One decode step of the framework's attention: appends k and v at `start`, attends over start + 1 positions."""
    from ppl_nn_b200 import ops
    batch = len(start)
    op = ops.MultiHeadCacheAttention(attention_param(hc, heads))
    kvlens = [s + 1 for s in start]
    out = op.forward(q, k, v, i64(range(batch + 1)), dev(starts_of(kvlens)), starts, i64(start), batch, 1, max(kvlens),
                     cache, scale)
    assert op.device_status() == 0
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("layout,page", [(0, 0), (3, 0), (0, 16), (3, 128)])
def test_a_drafted_step_is_a_run_of_decode_steps(gpu, pkg, layout, page):  # noqa: F811
    """History and drafted tokens are appended by the cache operator, the tree is attended to, an accepted path is moved
    to the front; the next decode step then gives, bit by bit, what it gives on a cache that never held the rest."""
    import torch
    from ppl_nn_b200 import ops
    rng = np.random.default_rng(layout + page)
    heads, kv_heads, dim = 8, 2, 128
    start, n = [37, 0, 200], [9, 4, 16]
    hc = HostCache(rng, [s + m + 1 for s, m in zip(start, n)], kv_heads, dim, layout, page)
    cache, scale, starts = dev(hc.cache), dev(hc.scale), dev(hc.starts)
    append = ops.KeyValueCache(ops.KeyValueCacheParam(**hc.param()))

    def put(to_cache, to_scale, counts, first, k, v):
        ends = [f + c for f, c in zip(first, counts)]
        append.forward(dev(k), dev(v), dev(starts_of(counts)), dev(starts_of(ends)), starts, i64(first), max(counts), max(ends),
                       to_cache, to_scale)

    def draw(total):
        return [rng.standard_normal((total, kv_heads, dim)).astype(np.float16) for _ in range(2)]

    hist_k, hist_v = draw(sum(start))
    tok_k, tok_v = draw(sum(n))
    put(cache, scale, start, [0] * 3, hist_k, hist_v)
    put(cache, scale, n, start, tok_k, tok_v)
    parents = sum([draw_parents(rng, m, "tree") for m in n], [])
    q = rng.standard_normal((sum(n), heads, dim)).astype(np.float16)
    tree = ops.TreeAttention(attention_param(hc, heads))
    got = tree.forward(dev(q), i64(parents), dev(starts_of(n)), starts, i64(start), max(n), max(s + m for s, m in zip(start, n)),
                       cache, scale)
    assert tree.device_status() == 0
    hc.cache, hc.scale = cache.cpu().numpy(), scale.cpu().numpy()
    hc.lens = [s + m for s, m in zip(start, n)]
    want, tol = tree_reference(hc, q, parents, start, n, heads, 0)
    assert np.all(np.abs(got.cpu().numpy() - want) <= tol)

    paths = []  # from a drafted token up to the root
    for b, first in enumerate(starts_of(n)[:-1]):
        at, path = n[b] - 1 - b, []
        while at >= 0:
            path.append(at)
            at = parents[first + at]
        paths.append(path[::-1])
    most = max(len(p) for p in paths) + 1
    kept = np.full((3, 1, most), -1, dtype=I64)
    for b, path in enumerate(paths):
        kept[b, 0, :len(path)] = path
    compact = ops.KeyValueCacheCompact(ops.KeyValueCacheParam(**hc.param()))
    compact.forward(dev(kept), starts, i64(start), i64(hc.lens), max(hc.lens), cache, scale)
    assert compact.device_status() == 0

    plain, plain_scale = torch.zeros_like(cache), torch.zeros_like(scale)
    put(plain, plain_scale, start, [0] * 3, hist_k, hist_v)
    rows = np.concatenate([[first + i for i in path] for first, path in zip(starts_of(n)[:-1], paths)]).astype(I64)
    put(plain, plain_scale, [len(p) for p in paths], start, tok_k[rows], tok_v[rows])
    now = [s + len(p) for s, p in zip(start, paths)]
    q1 = dev(rng.standard_normal((3, heads, dim)).astype(np.float16))
    k1, v1 = (dev(x) for x in draw(3))
    one = decode_output(hc, cache, scale, starts, heads, now, q1, k1, v1)
    two = decode_output(hc, plain, plain_scale, starts, heads, now, q1, k1, v1)
    assert torch.equal(one, two)


@pytest.mark.gpu
@pytest.mark.parametrize("layout,page", [(0, 0), (3, 48)])
def test_an_evicted_cache_decodes_like_one_of_the_kept_rows(gpu, pkg, layout, page):  # noqa: F811
    """Prompt window and decode steps add up weights, the highest stay, their rows move to the front with their weights;
    a decode step then gives what it gives on a cache into which the host gathered the same rows."""
    import torch
    from ppl_nn_b200 import ops
    rng = np.random.default_rng(layout)
    heads, kv_heads, dim = 8, 2, 64
    lens = [300, 90, 31]
    hc = HostCache(rng, [m + 1 for m in lens], kv_heads, dim, layout, page)
    hc.weight[:] = 0
    cache, scale, starts, weight = dev(hc.cache), dev(hc.scale), dev(hc.starts), dev(hc.weight)
    weigh = ops.AttentionWeight(attention_param(hc, heads))
    want, tol = np.zeros_like(hc.weight, dtype=np.float64), 0.0
    for n in ([16, 16, 16], [1, 1, 1]):  # the window at the end of the prompt, then a step
        q = rng.standard_normal((sum(n), heads, dim)).astype(np.float16)
        first = [m - x for m, x in zip(lens, n)]
        part, off = weight_reference(hc, q, first, n, heads, 0, True)
        want, tol = want + part, tol + off
        weigh.forward(dev(q), dev(starts_of(n)), starts, i64(first), max(n), max(lens), cache, scale, weight)
        assert weigh.device_status() == 0
    w = weight.cpu().numpy()
    # the second sum's rounding counts the first's weights as well
    assert np.all(np.abs(w - want) <= tol + 2.0 ** -23 * np.abs(want))
    budgets = [64, 90, 20]
    evict = ops.KeyValueCacheEvict(ops.KeyValueCacheEvictParam(**hc.param(), sink=2, recent=8))
    kept = evict.forward(weight, starts, i64(lens), i64(budgets), max(lens), max(budgets))
    compact = ops.KeyValueCacheCompact(ops.KeyValueCacheParam(**hc.param()))
    compact.forward(kept, starts, i64([0, 0, 0]), i64(lens), max(lens), cache, scale, weight)
    assert evict.device_status() == 0 and compact.device_status() == 0
    kept = kept.cpu().numpy()
    gathered, gathered_scale, gathered_w = hc.cache.copy(), hc.scale.copy(), w.copy()
    for b, m in enumerate(budgets):
        dst = hc.rows(b, np.arange(m))
        for h in range(kv_heads):
            assert (kept[b, h, :m] >= 0).all() and (kept[b, h, m:] == -1).all()
            src = hc.rows(b, kept[b, h, :m])
            if layout == 0:
                gathered[dst, :, :, h], gathered_scale[dst, :, :, h] = hc.cache[src, :, :, h], hc.scale[src, :, :, h]
            else:
                gathered[:, :, h, dst], gathered_scale[:, :, h, dst] = hc.cache[:, :, h, src], hc.scale[:, :, h, src]
            gathered_w[:, h, dst] = w[:, h, src]
            gathered_w[:, h, hc.rows(b, np.arange(m, lens[b]))] = 0
    assert np.array_equal(weight.cpu().numpy(), gathered_w)
    q1 = dev(rng.standard_normal((3, heads, dim)).astype(np.float16))
    k1, v1 = (dev(rng.standard_normal((3, kv_heads, dim)).astype(np.float16)) for _ in range(2))
    one = decode_output(hc, cache, scale, starts, heads, budgets, q1, k1, v1)
    two = decode_output(hc, dev(gathered), dev(gathered_scale), starts, heads, budgets, q1, k1, v1)
    assert torch.equal(one, two)


# ---- streams and captured calls ------------------------------------------------------------------------

class Step:
    """All four operators once, on inputs that stay where they are."""

    def __init__(self, seed, heads=8, kv_heads=2, dim=128):
        from ppl_nn_b200 import ops
        self.rng = np.random.default_rng(seed)
        self.heads, self.n = heads, [5, 1, 12]
        self.hc = hc = HostCache(self.rng, [700, 90, 330], kv_heads, dim, 3, 48)
        p = attention_param(hc, heads)
        self.tree, self.weigh = ops.TreeAttention(p), ops.AttentionWeight(p)
        self.evict = ops.KeyValueCacheEvict(ops.KeyValueCacheEvictParam(**hc.param(), sink=1, recent=9))
        self.compact = ops.KeyValueCacheCompact(ops.KeyValueCacheParam(**hc.param()))
        self.seq, self.starts, self.budgets = dev(starts_of(self.n)), dev(hc.starts), i64([100, 90, 40])
        self.base = i64([0, 0, 0])
        self.cache, self.scale, self.weight = dev(hc.cache), dev(hc.scale), dev(hc.weight)
        self.q = dev(self.rng.standard_normal((sum(self.n), heads, dim)).astype(np.float16))
        self.parents = i64(sum([draw_parents(self.rng, m, "tree") for m in self.n], []))
        self.lens = i64(hc.lens)
        self.start = self.lens - i64(self.n)

    def refill(self, seed):
        """New contents in the same places: other codes, queries, parents and lengths."""
        rng = np.random.default_rng(seed)
        lens = [int(rng.integers(m // 2, m + 1)) for m in self.hc.lens]
        for t, a in ((self.cache, rng.integers(-127, 128, size=self.hc.cache.shape, dtype=np.int8)),
                     (self.weight, rng.exponential(0.01, size=self.hc.weight.shape).astype(np.float32)),
                     (self.scale, self.hc.scale), (self.q, rng.standard_normal(tuple(self.q.shape)).astype(np.float16)),
                     (self.parents, np.array(sum([draw_parents(rng, m, "tree") for m in self.n], []))),
                     (self.lens, np.array(lens)), (self.start, np.array(lens) - np.array(self.n))):
            t.copy_(dev(a))

    def run(self):
        most = max(self.hc.lens)
        out = self.tree.forward(self.q, self.parents, self.seq, self.starts, self.start, 12, most, self.cache, self.scale)
        self.weigh.forward(self.q, self.seq, self.starts, self.start, 12, most, self.cache, self.scale, self.weight)
        kept = self.evict.forward(self.weight, self.starts, self.lens, self.budgets, most, 100)
        self.compact.forward(kept, self.starts, self.base, self.lens, most, self.cache, self.scale, self.weight)
        return [out, kept, self.cache, self.scale, self.weight]


@pytest.mark.gpu
def test_captured_steps_are_replayed_on_new_contents(gpu, pkg):  # noqa: F811
    import torch
    steps = [Step(1), Step(1)]
    # what the steps give in turn, eagerly
    want = []
    for seed in (11, 12, 13):
        steps[0].refill(seed)
        want.append([t.clone() for t in steps[0].run()])
    torch.cuda.synchronize()
    graphs, outs = [], []
    for s in steps:  # two graphs; the second's operators are the first's, too
        s.tree, s.weigh, s.evict, s.compact = steps[0].tree, steps[0].weigh, steps[0].evict, steps[0].compact
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(s.run())
        graphs.append(g)
    side = [torch.cuda.Stream(), torch.cuda.Stream()]
    for seeds in ((11, 12), (13, 11), (12, 13)):
        for s, seed in zip(steps, seeds):
            s.refill(seed)
        torch.cuda.synchronize()
        for g, stream in zip(graphs, side):  # at the same time
            with torch.cuda.stream(stream):
                g.replay()
        torch.cuda.synchronize()
        for out, seed in zip(outs, seeds):
            for x, y in zip(out, want[seed - 11]):
                assert torch.equal(x, y)


@pytest.mark.gpu
def test_steps_on_two_streams_share_the_operators(gpu, pkg):  # noqa: F811
    import torch
    alone = []
    for seed in (21, 22):
        s = Step(1)
        s.refill(seed)
        alone.append([t.clone() for t in s.run()])
    pair = [Step(1), Step(1)]
    pair[1].tree, pair[1].weigh, pair[1].evict, pair[1].compact = pair[0].tree, pair[0].weigh, pair[0].evict, pair[0].compact
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        for s, seed in zip(pair, (21, 22)):
            s.refill(seed)
        torch.cuda.synchronize()
        outs = []
        for s, stream in zip(pair, streams):
            with torch.cuda.stream(stream):
                outs.append(s.run())
        torch.cuda.synchronize()
        for out, want in zip(outs, alone):
            for x, y in zip(out, want):
                assert torch.equal(x, y)


@pytest.mark.gpu
def test_the_status_of_a_call_on_another_stream(gpu, pkg):  # noqa: F811
    """The status word is read behind the call's own stream, also from elsewhere and before anyone has waited for it."""
    import torch
    from ppl_nn_b200 import capi, ops
    rng = np.random.default_rng(1)
    hc = HostCache(rng, [40, 90], 2, 64)
    args = (dev(rng.standard_normal((7, 4, 64)).astype(np.float16)), i64([-1, 0, 9, -1, 0, 1, 2]), i64([0, 3, 7]), dev(hc.starts),
            i64([37, 86]), 4, 90, dev(hc.cache), dev(hc.scale))
    tree, side = ops.TreeAttention(attention_param(hc, 4)), torch.cuda.Stream()
    for fill in (0, 255):  # what the workspace may hold from before
        with torch.cuda.stream(side):
            del_me = torch.full((1 << 20,), fill, dtype=torch.uint8, device=gpu)
            del del_me
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            torch.cuda._sleep(100000000)
            tree.forward(*args)
        assert tree.device_status() == capi.DEV_PARENT_INVALID
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tree.forward(*args)
    with torch.cuda.stream(side):
        torch.cuda._sleep(100000000)
        graph.replay()
        assert tree.device_status() == capi.DEV_PARENT_INVALID


# ---- long caches -------------------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("layout,page", [(0, 0), (3, 0), (0, 128)])
def test_rows_beyond_two_to_the_31(gpu, pkg, layout, page):  # noqa: F811
    """Sequences at the end of a cache of 2.3 GB give what the same rows give in a small one, bit by bit."""
    import torch
    from ppl_nn_b200 import ops
    torch.manual_seed(layout + page)
    heads, kv_heads, dim, layers, tokens = 8, 4, 128, 4, 1 << 19
    lead = (tokens + 65536, layers, 2, kv_heads) if layout == 0 else (layers, 2, kv_heads, tokens + 65536)
    shift = 65536 + tokens - 4096  # the small cache's row 0
    big = torch.zeros(lead + (dim,), dtype=torch.int8, device=gpu)
    big_scale = torch.zeros(lead + (dim // 8,), dtype=torch.float16, device=gpu)
    assert big.numel() > 1 << 31
    rows = slice(shift, shift + 4096)
    cut = (rows,) if layout == 0 else (slice(None), slice(None), slice(None), rows)
    small = torch.randint(-127, 128, tuple(big[cut].shape), dtype=torch.int8, device=gpu)
    small_scale = torch.rand(tuple(big_scale[cut].shape), device=gpu).mul_(0.02).add_(0.005).half()
    big[cut], big_scale[cut] = small, small_scale
    n, start = [20, 3], [1500, 2000]
    starts = torch.tensor([100, 2000] if not page else [[i * 128 for i in order] for order in (range(0, 16), range(31, 15, -1))],
                          device=gpu, dtype=torch.int64)
    q = torch.randn(sum(n), heads, dim, device=gpu).half()
    parents = i64(sum([draw_parents(np.random.default_rng(3), m, "tree") for m in n], []))
    seq, first, lens = dev(starts_of(n)), i64(start), i64([s + m for s, m in zip(start, n)])
    geometry = dict(num_layer=layers, layer_idx=layers - 1, quant_bit=8, cache_mode=1 if page else 0, cache_layout=layout,
                    page_size=page or 128)
    p = ops.MultiHeadCacheAttentionParam(num_heads=heads, num_kv_heads=kv_heads, head_dim=dim, **geometry)
    res = []
    for cache, scale, at in ((small, small_scale, starts), (big, big_scale, starts + shift)):
        weight = torch.zeros(layers, kv_heads, cache.shape[0 if layout == 0 else 3], device=gpu)
        tree, weigh = ops.TreeAttention(p), ops.AttentionWeight(p)
        out = tree.forward(q, parents, seq, at, first, 20, 2003, cache, scale)
        weigh.forward(q, seq, at, first, 20, 2003, cache, scale, weight)
        last = torch.stack([q[19], q[22]])
        weigh.forward(last, i64([0, 1, 2]), at, lens - 1, 1, 2003, cache, scale, weight)
        evict = ops.KeyValueCacheEvict(ops.KeyValueCacheEvictParam(**geometry, sink=1, recent=4))
        kept = evict.forward(weight, at, lens, i64([700, 333]), 2003, 700)
        compact = ops.KeyValueCacheCompact(ops.KeyValueCacheParam(**geometry))
        compact.forward(kept, at, i64([0, 0]), lens, 2003, cache, scale, weight)
        assert [o.device_status() for o in (tree, weigh, evict, compact)] == [0] * 4
        part = cut if cache is big else (slice(None),)
        res.append([out, kept, cache[part].clone(), scale[part].clone(), weight[..., -4096:].clone()])
        if cache is big:  # nothing in front of the rows was touched
            rest = (slice(0, shift),) if layout == 0 else (slice(None), slice(None), slice(None), slice(0, shift))
            assert not cache[rest].any() and not weight[..., :-4096].any()
    for x, y in zip(*res):
        assert torch.equal(x, y)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["spread", "equal", "two values", "sampled high", "sorted"])
@pytest.mark.parametrize("n", [40000, 262144, 300001])
def test_select_of_long_lists(gpu, pkg, kind, n):  # noqa: F811
    """Lists beyond the shared memory, samples that mislead, and more equal weights than a list holds."""
    import torch
    from ppl_nn_b200 import ops
    rng = np.random.default_rng(n)
    budget, sink, recent = n // 3, 4, 100
    w = rng.exponential(1.0, size=n).astype(np.float32)
    if kind == "equal":
        w[:] = 0.25
    elif kind == "two values":
        w[:] = rng.integers(0, 2, size=n)
    elif kind == "sampled high":  # the sample's positions hold the highest weights
        have = n - recent - sink
        w[sink + (np.arange(4096) * (have / 4096)).astype(I64)] += 100
    elif kind == "sorted":
        w.sort()
    full = np.zeros((1, 1, n + 7), dtype=np.float32)
    full[0, 0, 3:3 + n] = w
    op = ops.KeyValueCacheEvict(ops.KeyValueCacheEvictParam(num_layer=1, layer_idx=0, quant_bit=8, cache_mode=0, cache_layout=0,
                                                            sink=sink, recent=recent))
    got = op.forward(dev(full), i64([3]), i64([n]), i64([budget]), n, budget)
    assert op.device_status() == 0
    cand = np.arange(sink, n - recent)
    order = cand[np.argsort(-w[cand], kind="stable")][:budget - sink - recent]
    want = np.sort(np.concatenate([np.arange(sink), order, np.arange(n - recent, n)]))
    assert torch.equal(got[0, 0].cpu(), torch.from_numpy(want))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["signs", "zeros", "few numbers", "infinities", "denormal", "negative", "nan at the cut", "all nan"])
@pytest.mark.parametrize("layout,page", [(0, 0), (3, 48)])
def test_select_of_long_lists_of_special_weights(gpu, pkg, kind, layout, page):  # noqa: F811
    """The bracket of the sample compares the weights themselves, the lists their keys: signs, zeros of both signs (which
    are equal), denormal numbers, infinities and NaN (below every number), with the cut on either side of them."""
    from ppl_nn_b200 import ops
    rng = np.random.default_rng(len(kind) + page)
    n, sink, recent = 70001, 4, 300
    hc = HostCache(rng, [n, 40000], 1, 64, layout, page)
    for b, m in enumerate(hc.lens):
        w = rng.standard_normal(m).astype(np.float32)
        pick = rng.random(m)
        if kind == "zeros":  # a third positive, the cut among the zeros of both signs
            w = np.where(pick < 0.33, np.abs(w), np.where(pick < 0.6, 0.0, -0.0)).astype(np.float32)
        elif kind == "few numbers":
            w[pick < 0.9] = np.nan
        elif kind == "infinities":
            w[pick < 0.3], w[pick > 0.7] = np.inf, -np.inf
        elif kind == "denormal":
            w = (w * 1e-40).astype(np.float32)
        elif kind == "negative":
            w = -np.abs(w)
            w[pick < 0.2] = -0.0
        elif kind == "nan at the cut":
            w[pick < 0.5] = np.nan
            w[pick > 0.9] = np.inf
        elif kind == "all nan":
            w[:] = np.nan
        hc.weight[0, 0, hc.rows(b, np.arange(m))] = w
    op = ops.KeyValueCacheEvict(ops.KeyValueCacheEvictParam(**hc.param(), sink=sink, recent=recent))
    for budget in (sink + recent + 1, 6000, 20000, 30304, 39000):
        kept = op.forward(dev(hc.weight), dev(hc.starts), i64(hc.lens), i64([budget, budget - 7]), n, budget).cpu().numpy()
        assert op.device_status() == 0
        for b, m in enumerate(hc.lens):
            k = budget - 7 * b
            w = hc.weight[0, 0, hc.rows(b, np.arange(m))].astype(np.float64)
            s, r = min(sink, k - min(recent, k)), min(recent, k)
            cand = np.arange(s, m - r)
            order = cand[np.lexsort((cand, -np.where(np.isnan(w), 0, w)[cand], np.isnan(w)[cand]))][:k - r - s]
            want = np.sort(np.concatenate([np.arange(s), order, np.arange(m - r, m)]))
            assert np.array_equal(kept[b, 0, :k], want) and (kept[b, 0, k:] == -1).all()


# ---- forms of the weights and of the tree --------------------------------------------------------------

MORE_WEIGHT_CASES = [
    # heads, kv heads, dim, start, n, layout, page, layers, layer, causal: 1, 2, 3..4, 5..8, 9..16, 17..32 and many rows, both
    # head sizes
    (4, 4, 128, [0, 31, 600], [1, 1, 1], 0, 0, 1, 0, True),
    (3, 3, 64, [5, 1023], [1, 1], 3, 48, 1, 0, True),
    (4, 2, 128, [0, 16, 1500], [1, 1, 1], 3, 0, 1, 0, True),
    (4, 2, 64, [47, 200], [1, 1], 0, 16, 1, 0, True),
    (2, 2, 64, [0, 100, 33], [2, 1, 0], 0, 0, 2, 1, True),
    (2, 2, 128, [64, 9], [2, 2], 0, 0, 1, 0, False),
    (8, 2, 64, [15, 700], [1, 1], 0, 0, 1, 0, True),
    (6, 2, 64, [300, 2], [1, 1], 3, 128, 1, 0, True),
    (2, 1, 128, [0, 515], [2, 2], 0, 16, 1, 0, True),
    (16, 2, 128, [0, 900], [1, 1], 0, 0, 1, 0, True),
    (5, 1, 128, [63], [1], 3, 0, 1, 0, True),
    (9, 1, 64, [64, 0], [1, 1], 0, 0, 1, 0, True),
    (8, 2, 128, [300, 0, 77], [3, 4, 1], 0, 0, 1, 0, True),
    (4, 1, 64, [50, 600], [4, 3], 3, 48, 1, 0, False),
    (8, 1, 128, [700, 3], [4, 3], 3, 0, 1, 0, True),
    (8, 2, 64, [100, 1030], [5, 2], 0, 16, 1, 0, True),
    (7, 1, 128, [0, 2000], [1, 3], 0, 0, 2, 0, False),
    (32, 4, 64, [0, 1100], [40, 17], 0, 0, 1, 0, True),
    (32, 4, 128, [980, 3], [33, 2], 3, 64, 2, 0, False),
    (4, 1, 128, [2040], [300], 0, 128, 1, 0, True),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", MORE_WEIGHT_CASES, ids=str)
def test_attention_weight_forms(gpu, pkg, case):  # noqa: F811
    from ppl_nn_b200 import ops
    heads, kv_heads, dim, start, n, layout, page, layers, layer, causal = case
    rng = np.random.default_rng(sum(start) + dim)
    hc = HostCache(rng, [s + m for s, m in zip(start, n)], kv_heads, dim, layout, page, layers)
    q = rng.standard_normal((sum(n), heads, dim)).astype(np.float16)
    want, tol = weight_reference(hc, q, start, n, heads, layer, causal)
    op = ops.AttentionWeight(attention_param(hc, heads, layer, is_causal=causal))
    for max_n, max_len in ((max(n), hc.max_len), (max(n), hc.max_len + (0 if page else 1000))):
        weight, cache, scale = dev(hc.weight), dev(hc.cache), dev(hc.scale)
        op.forward(dev(q), dev(starts_of(n)), dev(hc.starts), i64(start), max_n, max_len, cache, scale, weight)
        assert op.device_status() == 0
        got = weight.cpu().numpy()
        assert np.all(np.abs(got - want) <= tol), float((np.abs(got - want) / tol).max())
        assert np.array_equal(cache.cpu().numpy(), hc.cache) and np.array_equal(scale.cpu().numpy(), hc.scale)
    # a larger bound on the query tokens picks another form, not another result
    weight = dev(hc.weight)
    op.forward(dev(q), dev(starts_of(n)), dev(hc.starts), i64(start), max(n) + 9, hc.max_len, dev(hc.cache), dev(hc.scale), weight)
    assert op.device_status() == 0
    assert np.all(np.abs(weight.cpu().numpy() - want) <= tol)


@pytest.mark.gpu
def test_weights_of_sequences_that_share_rows_add_up(gpu, pkg):  # noqa: F811
    """Two sequences over the same cache rows: both add to them (a shared prefix)."""
    from ppl_nn_b200 import ops
    rng = np.random.default_rng(8)
    hc = HostCache(rng, [200, 200], 2, 64)
    hc.starts[1] = hc.starts[0]
    for n in ([1, 1], [9, 9]):
        start = [200 - m for m in n]
        q = rng.standard_normal((sum(n), 4, 64)).astype(np.float16)
        want, tol = weight_reference(hc, q, start, n, 4, 0, True)
        weight = dev(hc.weight)
        ops.AttentionWeight(attention_param(hc, 4)).forward(dev(q), dev(starts_of(n)), dev(hc.starts), i64(start), max(n), 200,
                                                             dev(hc.cache), dev(hc.scale), weight)
        # one more rounding than the reference counts: two additions to a row
        assert np.all(np.abs(weight.cpu().numpy() - want) <= tol + 2.0 ** -23 * np.abs(want))


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv_heads,dim,n", [(8, 2, 128, [3, 12]), (8, 2, 64, [5, 1]), (8, 1, 128, [40, 9]), (16, 1, 64, [17, 30])])
def test_keys_of_a_tree_are_not_rounded(gpu, pkg, heads, kv_heads, dim, n):  # noqa: F811
    """One group of channels whose keys are 40 times the others', as after outlying activations: scores of tens, which a
    rounding of the keys to fp16 would move by hundredths.

    A score is a sum of 2 Dh exact products in fp32: Dh / 8 tensor-core instructions, each off by at most 2^-22 of the
    products' magnitudes; that is an error of the exponent, of a weight and of the normaliser.  Weights, values and the
    output are rounded to fp16 (2^-11), weights below its normal range by 2^-25 of the largest; 2^-16 covers the
    exponentials and the sums."""
    rng = np.random.default_rng(dim + n[0])
    start, u = [700, 90], 2.0 ** -11
    hc = HostCache(rng, [s + m for s, m in zip(start, n)], kv_heads, dim)
    hc.scale[:, :, 0, :, 3] = (hc.scale[:, :, 0, :, 3].astype(np.float32) * 40).astype(np.float16)
    q = rng.standard_normal((sum(n), heads, dim)).astype(np.float16)
    parents = sum([draw_parents(rng, m, "tree") for m in n], [])
    want, _ = tree_reference(hc, q, parents, start, n, heads, 0)
    tol, first, group = np.zeros(q.shape), 0, heads // kv_heads
    for b, m in enumerate(n):
        rows = hc.rows(b, np.arange(start[b] + m))
        for g in range(kv_heads):
            k, v = hc.values(0, 0, g, rows), hc.values(1, 0, g, rows)
            for i in range(first, first + m):
                for h in range(g * group, (g + 1) * group):
                    x = q[i, h].astype(np.float64)
                    off = (dim / 8) * 2.0 ** -22 * (np.abs(k) @ np.abs(x)).max() / np.sqrt(dim)
                    tol[i, h] = (np.abs(v).max(0) * (2 * off + 2 * u + 2.0 ** -16) + u * np.abs(want[i, h])
                                 + 2 * len(k) * 2.0 ** -25 * np.abs(v).max())
        first += m
    got, status = run_tree(hc, q, parents, start, n, heads, 0)
    assert status == 0
    assert np.all(np.abs(got - want) <= tol), float((np.abs(got - want) / tol).max())


class OutsideCache(HostCache):
    """A cache some of whose positions name rows outside it: keys and values of zeros, without a weight of their own."""

    def values(self, which, layer, head, rows):
        inside = (rows >= 0) & (rows < self.max_tokens)
        out = np.zeros((len(rows), self.dim))
        out[inside] = super().values(which, layer, head, rows[inside])
        return out


@pytest.mark.gpu
@pytest.mark.parametrize("n", [[1, 1], [4, 2], [40, 9]])  # 2, 8 and 80 query rows
@pytest.mark.parametrize("layout,page,where", [(0, 0, "beyond"), (3, 0, "before"), (0, 16, "beyond"), (3, 64, "before"), (0, 48, "beyond")])
def test_rows_outside_the_cache_count_as_zeros(gpu, pkg, n, layout, page, where):  # noqa: F811
    """Reported, and read as zeros, as decode and prefill read them: with a score of 0."""
    from ppl_nn_b200 import capi, ops
    rng = np.random.default_rng(page + n[0])
    start, heads = [150, 333], 4
    hc = OutsideCache(rng, [s + m for s, m in zip(start, n)], 2, 64, layout, page)
    while page and (hc.starts == hc.max_tokens - page).any():  # the last page is to be nobody's
        hc = OutsideCache(rng, [s + m for s, m in zip(start, n)], 2, 64, layout, page)
    hc.scale[:] = 0.002  # scores of a few tenths: the rows outside weigh as much as the others
    if page:
        hc.starts[1, 2] = hc.max_tokens + 5 if where == "beyond" else -page
        hc.starts[0, 1] = hc.max_tokens - 16 if page > 16 else 1 << 40  # a page that ends outside, where it is long enough
    else:
        hc.starts[1] = hc.max_tokens - 200 if where == "beyond" else -7
    q = rng.standard_normal((sum(n), heads, 64)).astype(np.float16)
    args = (dev(starts_of(n)), dev(hc.starts), i64(start), max(n), hc.max_len, dev(hc.cache), dev(hc.scale))
    parents = sum([draw_parents(rng, m, "tree") for m in n], [])
    rows = hc.rows
    if where == "before" and not page:  # no position of a sequence that starts before the cache has a row
        hc.rows = lambda b, p: rows(b, p) if b == 0 else np.full(len(p), -1)
    tree = ops.TreeAttention(attention_param(hc, heads))
    got = tree.forward(dev(q), i64(parents), *args).cpu().numpy()
    assert tree.device_status() == capi.DEV_ROW_OUT_OF_RANGE
    want, tol = tree_reference(hc, q, parents, start, n, heads, 0)
    assert np.all(np.abs(got - want) <= tol)
    # the reference of the weights adds to the row of each position: those outside go behind the cache
    named, held = hc.rows, hc.weight
    hc.weight = np.concatenate([held, np.zeros((1, 2, 1 << 10), dtype=np.float32)], axis=-1)
    hc.rows = lambda b, p: np.where((named(b, p) >= 0) & (named(b, p) < hc.max_tokens), named(b, p), hc.max_tokens + np.asarray(p))
    want, tol = weight_reference(hc, q, start, n, heads, 0, True)
    weight, weigh = dev(held), ops.AttentionWeight(attention_param(hc, heads))
    weigh.forward(dev(q), *args, weight)
    assert weigh.device_status() == capi.DEV_ROW_OUT_OF_RANGE
    want, tol = want[..., :hc.max_tokens], tol[..., :hc.max_tokens]
    assert np.all(np.abs(weight.cpu().numpy() - want) <= tol)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [[3, 1], [40, 9]])
def test_tokens_behind_the_last_sequence_are_padding(gpu, pkg, n):  # noqa: F811
    """A padded batch: queries behind seqstarts[-1] are not read, their outputs stay as they were."""
    import torch
    from ppl_nn_b200 import ops
    rng = np.random.default_rng(n[0])
    start = [130, 7]
    hc = HostCache(rng, [s + m for s, m in zip(start, n)], 2, 64)
    q = rng.standard_normal((sum(n) + 5, 8, 64)).astype(np.float16)
    q[sum(n):] = np.nan
    args = (dev(q), dev(starts_of(n)), dev(hc.starts), i64(start), max(n), hc.max_len, dev(hc.cache), dev(hc.scale))
    parents = sum([draw_parents(rng, m, "tree") for m in n], [])
    want, tol = tree_reference(hc, q[:sum(n)], parents, start, n, 8, 0)
    out = torch.full(q.shape, 7.0, dtype=torch.float16, device=gpu)
    tree = ops.TreeAttention(attention_param(hc, 8))
    tree.forward(args[0], i64(parents + [99] * 5), *args[1:], attn_output=out)
    assert tree.device_status() == 0
    got = out.cpu().numpy()
    assert np.all(np.abs(got[:sum(n)] - want) <= tol) and (got[sum(n):] == 7).all()
    want, tol = weight_reference(hc, q[:sum(n)], start, n, 8, 0, True)
    weight = dev(hc.weight)
    weigh = ops.AttentionWeight(attention_param(hc, 8))
    weigh.forward(*args, weight)
    assert weigh.device_status() == 0 and np.all(np.abs(weight.cpu().numpy() - want) <= tol)


@pytest.mark.gpu
def test_the_largest_tree(gpu, pkg):  # noqa: F811
    rng = np.random.default_rng(5)
    start, n = [70, 3], [1024, 129]
    hc = HostCache(rng, [s + m for s, m in zip(start, n)], 1, 64)
    q = rng.standard_normal((sum(n), 2, 64)).astype(np.float16)
    parents = draw_parents(rng, 1024, "tree") + draw_parents(rng, 129, "star")
    want, tol = tree_reference(hc, q, parents, start, n, 2, 0)
    got, status = run_tree(hc, q, parents, start, n, 2, 0)
    assert status == 0
    assert np.all(np.abs(got - want) <= tol), float((np.abs(got - want) / tol).max())
    again, _ = run_tree(hc, q, parents, start, n, 2, 0)
    assert np.array_equal(again, got)
