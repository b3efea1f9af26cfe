"""The operators around the INT8 cache -- accumulated attention weight, eviction, compaction -- against plain numpy
in 64 bits.  Refusals are checked on the host, without a GPU."""
import ctypes
import math

import numpy as np
import pytest

GROUP = 8


# ---- a cache and its rows, on the host -----------------------------------------------------------

class HostCache:
    """Codes, scales and weights of a batch, and the cache row of every position."""

    def __init__(self, rng, lens, heads, dim, layout=0, page=0, layers=1, slack=5):
        self.lens, self.heads, self.dim, self.layout, self.page, self.layers = list(lens), heads, dim, layout, page, layers
        if page:
            pages = [-(-n // page) for n in self.lens]
            order = rng.permutation(sum(pages) + 1)
            self.starts = np.zeros((len(self.lens), max(max(pages, default=1), 1)), dtype=np.int64)
            at = 0
            for b, n in enumerate(pages):
                self.starts[b, :n] = order[at:at + n] * page
                at += n
            self.max_tokens = (sum(pages) + 1) * page
        else:
            self.starts = np.cumsum([slack] + [n + slack for n in self.lens])[:-1].astype(np.int64)
            self.max_tokens = int(sum(self.lens) + slack * (len(self.lens) + 1))
        lead = (self.max_tokens, layers, 2, heads) if layout == 0 else (layers, 2, heads, self.max_tokens)
        self.cache = rng.integers(-127, 128, size=lead + (dim,), dtype=np.int8)
        self.scale = rng.uniform(0.004, 0.03, size=lead + (dim // GROUP,)).astype(np.float16)
        self.weight = rng.exponential(0.01, size=(layers, heads, self.max_tokens)).astype(np.float32)

    def rows(self, b, positions):
        p = np.asarray(positions, dtype=np.int64)
        return self.starts[b, p // self.page] + p % self.page if self.page else self.starts[b] + p

    def values(self, which, layer, head, rows):
        if self.layout == 0:
            c, s = self.cache[rows, layer, which, head], self.scale[rows, layer, which, head]
        else:
            c, s = self.cache[layer, which, head, rows], self.scale[layer, which, head, rows]
        return c.astype(np.float64) * np.repeat(s.astype(np.float64), GROUP, axis=-1)

    def param(self, layer_idx=0):
        return dict(num_layer=self.layers, layer_idx=layer_idx, quant_bit=8, cache_mode=1 if self.page else 0,
                    cache_layout=self.layout, page_size=self.page or 128)

    @property
    def max_len(self):
        return max(self.lens, default=0)


def dev(a, device="cuda"):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).to(device)


def starts_of(counts):
    return np.concatenate([[0], np.cumsum(counts)]).astype(np.int64)


@pytest.fixture(scope="module")
def gpu(built_lib):
    import torch
    if not torch.cuda.is_available():
        pytest.fail("a test marked gpu ran without a CUDA device")
    assert built_lib.device_ready(), "the CUDA library has no sm_100a code for this device"
    return torch.device("cuda:0")


# ---- refusals on the host ------------------------------------------------------------------------

def _params(lib, capi, **kw):
    p = capi.AttnParams()
    p.num_heads, p.num_kv_heads, p.head_dim, p.is_causal = 32, 8, 128, 1
    p.num_layer, p.layer_idx, p.quant_bit, p.quant_group = 4, 1, 8, 8
    p.page_size = 128
    p.batch, p.max_seqlen, p.max_kvlen, p.total_tokens, p.max_tokens = 4, 2, 600, 8, 1 << 16
    for k, v in kw.items():
        setattr(p, k, v)
    assert lib.fill_cache_strides(p) == capi.SUCCESS
    return p


FAKE = ctypes.c_void_p(4096)


def _weight_call(lib, p, q=FAKE, seq=FAKE, start=FAKE, cache=FAKE, scale=FAKE, w=FAKE, ws=FAKE, n=1 << 40):
    return lib.attn_weight_accumulate(p, q, seq, FAKE, start, cache, scale, w, ws, n, None)


def _select_call(lib, p, w=FAKE, lens=FAKE, sink=0, recent=0, most=16, kept=FAKE, ws=FAKE, n=1 << 40):
    return lib.kv_evict_select(p, w, FAKE, lens, FAKE, sink, recent, most, kept, ws, n, None)


def _compact_call(lib, p, kept=FAKE, heads=8, most=16, base=FAKE, layers=1, cache=FAKE, scale=FAKE, w=None, ws=FAKE,
                  n=1 << 40):
    return lib.kv_compact(p, kept, heads, most, base, FAKE, FAKE, layers, cache, scale, w, ws, n, None)


@pytest.mark.parametrize("call", [_weight_call, _select_call, _compact_call])
@pytest.mark.parametrize("field,value,expect", [
    ("quant_bit", 4, "RC_UNSUPPORTED"), ("head_dim", 96, "RC_UNSUPPORTED"), ("cache_layout", 1, "RC_UNSUPPORTED"),
    ("num_kv_heads", 5, "RC_INVALID_VALUE"), ("layer_idx", 4, "RC_INVALID_VALUE"), ("max_tokens", 0, "RC_INVALID_VALUE"),
    ("max_kvlen", 1 << 31, "RC_UNSUPPORTED"), ("batch", 65536, "RC_UNSUPPORTED"), ("batch", -1, "RC_INVALID_VALUE"),
])
def test_attributes_are_refused(built_lib, pkg, call, field, value, expect):
    from ppl_nn_b200 import capi
    p = _params(built_lib, capi)
    setattr(p, field, value)
    assert built_lib.status_str(call(built_lib, p)) == expect


@pytest.mark.parametrize("call,kw,expect", [
    (_weight_call, dict(scale=None), "RC_UNSUPPORTED"),
    (_weight_call, dict(w=None), "RC_NOT_FOUND"),
    (_weight_call, dict(q=ctypes.c_void_p(4104)), "RC_INVALID_VALUE"),
    (_weight_call, dict(start=ctypes.c_void_p(4100)), "RC_INVALID_VALUE"),
    (_select_call, dict(sink=-1), "RC_INVALID_VALUE"),
    (_select_call, dict(recent=-1), "RC_INVALID_VALUE"),
    (_select_call, dict(most=-1), "RC_INVALID_VALUE"),
    (_select_call, dict(kept=None), "RC_NOT_FOUND"),
    (_select_call, dict(lens=ctypes.c_void_p(4100)), "RC_INVALID_VALUE"),
    (_compact_call, dict(heads=4), "RC_INVALID_VALUE"),
    (_compact_call, dict(layers=4), "RC_INVALID_VALUE"),
    (_compact_call, dict(layers=0), "RC_INVALID_VALUE"),
    (_compact_call, dict(most=-1), "RC_INVALID_VALUE"),
    (_compact_call, dict(scale=None), "RC_UNSUPPORTED"),
    (_compact_call, dict(kept=None), "RC_NOT_FOUND"),
    (_compact_call, dict(cache=ctypes.c_void_p(4100)), "RC_INVALID_VALUE"),
])
def test_arguments_are_refused(built_lib, pkg, call, kw, expect):
    from ppl_nn_b200 import capi
    assert built_lib.status_str(call(built_lib, _params(built_lib, capi), **kw)) == expect


def test_empty_calls_and_missing_device(built_lib, pkg):
    import torch
    from ppl_nn_b200 import capi
    empty = _params(built_lib, capi, batch=0, total_tokens=0)
    assert _weight_call(built_lib, empty, q=None, w=None) == capi.SUCCESS
    assert _select_call(built_lib, empty, w=None, kept=None) == capi.SUCCESS
    assert _compact_call(built_lib, empty, cache=None, base=None) == capi.SUCCESS
    if not torch.cuda.is_available():
        p = _params(built_lib, capi)
        for call in (_weight_call, _select_call, _compact_call):
            assert built_lib.status_str(call(built_lib, p)) == "RC_NO_DEVICE_CODE"


def test_workspace_sizes(built_lib, pkg):
    from ppl_nn_b200 import capi
    assert built_lib.kv_evict_workspace_size(_params(built_lib, capi)) == (capi.SUCCESS, 256)
    sizes = [built_lib.kv_compact_workspace_size(_params(built_lib, capi), heads, most, layers)
             for heads, most, layers in ((1, 0, 1), (1, 8, 1), (8, 64, 1), (8, 640, 3))]
    assert all(rc == capi.SUCCESS and n % 256 == 0 for rc, n in sizes)
    assert [n for _, n in sizes] == sorted(n for _, n in sizes)
    rc, _ = built_lib.kv_compact_workspace_size(_params(built_lib, capi), 3, 8, 1)
    assert built_lib.status_str(rc) == "RC_INVALID_VALUE"
    rc, n = built_lib.attn_weight_workspace_size(_params(built_lib, capi))
    assert rc == capi.SUCCESS and n % 256 == 0 and n > 8 * 8 * 32
    rc, more = built_lib.attn_weight_workspace_size(_params(built_lib, capi, max_kvlen=60000))
    assert rc == capi.SUCCESS and more > n


# ---- accumulated attention weight ------------------------------------------------------------------

def weight_reference(hc, q, start, n, heads, layer, causal):
    """New weights, and how far a result may be off each, in 64 bits.

    A score is a sum of 2 Dh exact products (key and remainder, each with the fp16 query) in fp32 accumulators: Dh / 8
    tensor-core instructions, each off by at most 2^-22 of the sum of the products' magnitudes A (two units in the
    last place, for alignment and truncation); scaled by 1/sqrt(Dh) that is an absolute error of the exponent, and
    enters a weight once by its own score and once, at worst, by the row's normaliser.  Exponentials are off by 2^-22
    each, the products and sums behind them by 2^-24 a step; 2^-18 covers them (64 steps).  The addition to the old
    weight rounds once more, and underflow is below 2^-126."""
    group = heads // hc.heads
    out, tol = hc.weight.astype(np.float64), np.zeros(hc.weight.shape)
    first = 0
    for b in range(len(hc.lens)):
        rows = hc.rows(b, np.arange(start[b] + n[b]))
        for g in range(hc.heads):
            k = hc.values(0, layer, g, rows)
            for i in range(n[b]):
                see = start[b] + i + 1 if causal else start[b] + n[b]
                for h in range(group):
                    x = q[first + i, g * group + h].astype(np.float64)
                    s = k[:see] @ x / math.sqrt(hc.dim)
                    p = np.exp(s - s.max())
                    p /= p.sum()
                    big = (np.abs(k[:see]) @ np.abs(x)).max() / math.sqrt(hc.dim)
                    out[layer, g, rows[:see]] += p
                    tol[layer, g, rows[:see]] += p * (2 * (hc.dim / 8) * 2.0 ** -22 * big + 2.0 ** -18)
        first += n[b]
    return out, tol + 2.0 ** -23 * np.abs(out) + 2.0 ** -120


WEIGHT_CASES = [
    # heads, kv heads, dim, start, n, layout, page, layers, layer, causal
    (8, 8, 64, [0, 15, 16, 511], [1, 1, 1, 1], 0, 0, 1, 0, True),
    (8, 2, 128, [0, 1, 31, 512, 1030], [1, 1, 1, 1, 1], 0, 0, 1, 0, True),
    (8, 1, 64, [700, 17], [1, 1], 3, 0, 2, 1, True),
    (12, 4, 128, [513, 40], [1, 1], 0, 16, 1, 0, True),
    (32, 8, 128, [0, 100, 490], [7, 1, 33], 0, 0, 3, 1, True),
    (6, 2, 64, [0, 0, 20], [1, 0, 5], 3, 48, 1, 0, True),
    (16, 2, 128, [37, 600], [11, 3], 0, 48, 1, 0, False),
    (10, 2, 128, [5, 1000], [20, 2], 3, 0, 1, 0, True),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", WEIGHT_CASES, ids=str)
def test_attention_weight(gpu, pkg, case):
    from ppl_nn_b200 import ops
    heads, kv_heads, dim, start, n, layout, page, layers, layer, causal = case
    rng = np.random.default_rng(len(str(case)))
    hc = HostCache(rng, [s + m for s, m in zip(start, n)], kv_heads, dim, layout, page, layers)
    q = rng.standard_normal((sum(n), heads, dim)).astype(np.float16)
    want, tol = weight_reference(hc, q, start, n, heads, layer, causal)
    op = ops.AttentionWeight(ops.MultiHeadCacheAttentionParam(num_heads=heads, num_kv_heads=kv_heads, head_dim=dim,
                                                              is_causal=causal, **hc.param(layer)))
    weight = dev(hc.weight)
    args = (dev(q), dev(starts_of(n)), dev(hc.starts), dev(np.array(start, dtype=np.int64)), max(n), hc.max_len,
            dev(hc.cache), dev(hc.scale))
    assert op.forward(*args, weight) is weight
    assert op.device_status() == 0
    got = weight.cpu().numpy()
    assert np.all(np.abs(got - want) <= tol), float((np.abs(got - want) - tol).max())
    # rows of no sequence, and the other layers, stay as they were
    assert np.array_equal(got[tol <= 2.0 ** -23 * np.abs(want) + 2.0 ** -119], hc.weight[tol <= 2.0 ** -23 * np.abs(want) + 2.0 ** -119])
    # the same call on the same weights gives the same bits
    again = dev(hc.weight)
    op.forward(*args, again)
    assert np.array_equal(again.cpu().numpy(), got)


@pytest.mark.gpu
def test_attention_weight_of_nan_behind_the_sequence_and_bad_rows(gpu, pkg):
    """Codes of positions that no query may see do not matter; a row outside the cache is reported and skipped."""
    from ppl_nn_b200 import capi, ops
    rng = np.random.default_rng(3)
    hc = HostCache(rng, [40, 90], 2, 64)
    q = rng.standard_normal((2, 4, 64)).astype(np.float16)
    for b in range(2):  # everything behind the sequences is NaN
        hc.scale[hc.starts[b] + hc.lens[b]:(hc.starts[b + 1] if b == 0 else None)] = np.nan
    want, tol = weight_reference(hc, q, [39, 89], [1, 1], 4, 0, True)
    op = ops.AttentionWeight(ops.MultiHeadCacheAttentionParam(num_heads=4, num_kv_heads=2, head_dim=64, **hc.param()))
    weight = dev(hc.weight)
    start = np.array([39, 89], dtype=np.int64)
    args = [dev(q), dev(starts_of([1, 1])), dev(hc.starts), dev(start), 1, 90, dev(hc.cache), dev(hc.scale)]
    op.forward(*args, weight)
    assert op.device_status() == 0
    assert np.all(np.abs(weight.cpu().numpy() - want) <= tol)
    args[2] = dev(np.array([hc.starts[0], hc.max_tokens - 50], dtype=np.int64))
    op.forward(*args, dev(hc.weight))
    assert op.device_status() & capi.DEV_ROW_OUT_OF_RANGE


# ---- eviction --------------------------------------------------------------------------------------

def select_reference(w, n, budget, sink, recent):
    """Kept positions of one list of weights."""
    k = min(budget, n)
    r = min(recent, k)
    s = min(sink, k - r)
    rank = np.where(np.isnan(w[:n]), -np.inf, w[:n])
    cand = np.arange(s, n - r)
    # NaN below everything, -inf too; ties to the lowest position
    order = sorted(cand, key=lambda j: (0 if not np.isnan(w[j]) else 1, -rank[j], j))
    return sorted(list(range(s)) + order[:k - r - s] + list(range(n - r, n)))


@pytest.mark.gpu
@pytest.mark.parametrize("layout,page", [(0, 0), (3, 48), (0, 16)])
@pytest.mark.parametrize("values", ["spread", "ties", "signs", "extremes"])
@pytest.mark.parametrize("budget,sink,recent", [(1, 0, 0), (0, 3, 3), (37, 4, 9), (10, 8, 8), (100000, 1, 1), (500, 0, 0)])
def test_evict_select(gpu, pkg, layout, page, values, budget, sink, recent):
    from ppl_nn_b200 import ops
    rng = np.random.default_rng(budget + sink)
    lens = [1, 2, 17, 300, 1024, 2500, 0]
    hc = HostCache(rng, lens, 3, 64, layout, page, layers=2)
    w = hc.weight
    if values == "ties":
        w[:] = rng.integers(0, 3, size=w.shape)
    elif values == "signs":
        w[:] = rng.standard_normal(w.shape)
        w[rng.random(w.shape) < 0.2] = -0.0
        w[rng.random(w.shape) < 0.2] = 0.0
    elif values == "extremes":
        pick = rng.random(w.shape)
        w[pick < 0.3] = np.nan
        w[(pick > 0.3) & (pick < 0.5)] = np.inf
        w[(pick > 0.5) & (pick < 0.6)] = -np.inf
        w[(pick > 0.6) & (pick < 0.7)] = 1e-42
    budgets = np.minimum(np.array([budget] * len(lens)), 2600)
    budgets[3] = max(0, budgets[3] - 1)
    most = int(budgets.max()) + 2
    op = ops.KeyValueCacheEvict(ops.KeyValueCacheEvictParam(**hc.param(1), sink=sink, recent=recent))
    kept = op.forward(dev(w), dev(hc.starts), dev(np.array(lens, dtype=np.int64)), dev(budgets), hc.max_len, most)
    assert op.device_status() == 0
    kept = kept.cpu().numpy()
    assert kept.shape == (len(lens), 3, most)
    for b, n in enumerate(lens):
        rows = hc.rows(b, np.arange(n))
        for g in range(3):
            want = select_reference(w[1, g, rows], n, int(budgets[b]), sink, recent)
            assert list(kept[b, g, :len(want)]) == want, (b, g)
            assert (kept[b, g, len(want):] == -1).all()


@pytest.mark.gpu
def test_evict_select_long_list_and_cut_length(gpu, pkg):
    from ppl_nn_b200 import capi, ops
    rng = np.random.default_rng(5)
    lens = [70001]
    hc = HostCache(rng, lens, 1, 64)
    hc.weight[0, 0, rng.integers(0, hc.max_tokens, 30000)] = 0.25  # many equal ones around the cut
    w = hc.weight[0, 0, hc.rows(0, np.arange(70001))]
    op = ops.KeyValueCacheEvict(ops.KeyValueCacheEvictParam(**hc.param(), sink=4, recent=1000))
    for budget in (1005, 12345, 40000, 70000):
        kept = op.forward(dev(hc.weight), dev(hc.starts), dev(np.array(lens)), dev(np.array([budget])), 70001, budget)
        assert list(kept[0, 0].cpu().numpy()) == select_reference(w, 70001, budget, 4, 1000)
        assert op.device_status() == 0
    kept = op.forward(dev(hc.weight), dev(hc.starts), dev(np.array(lens)), dev(np.array([2000])), 5000, 2000)
    assert op.device_status() == capi.DEV_LENGTH_CLAMPED
    assert list(kept[0, 0].cpu().numpy()) == select_reference(w, 5000, 2000, 4, 1000)


@pytest.mark.gpu
def test_evict_select_reports_negative_lengths(gpu, pkg):
    from ppl_nn_b200 import capi, ops
    rng = np.random.default_rng(6)
    hc = HostCache(rng, [50, 3000], 2, 64)
    op = ops.KeyValueCacheEvict(ops.KeyValueCacheEvictParam(**hc.param(), sink=1, recent=2))
    for most in (50, 3000):  # short and long lists
        kept = op.forward(dev(hc.weight), dev(hc.starts), dev(np.array([-1, most])), dev(np.array([7, 9])), most, 9).cpu().numpy()
        assert op.device_status() == capi.DEV_LENGTH_CLAMPED
        assert (kept[0] == -1).all()
        for g in range(2):
            assert list(kept[1, g]) == select_reference(hc.weight[0, g, hc.rows(1, np.arange(most))], most, 9, 1, 2)


# ---- compaction ------------------------------------------------------------------------------------

def compact_reference(hc, kept, base, first_layer, layers, with_weight, lens=None):
    cache, scale, weight = hc.cache.copy(), hc.scale.copy(), hc.weight.copy()
    for b in range(len(hc.lens)):
        for g in range(hc.heads):
            mine = kept[b, g if kept.shape[1] > 1 else 0]
            mine = mine[:np.argmax(mine < 0)] if (mine < 0).any() else mine
            src, dst = hc.rows(b, base[b] + mine), hc.rows(b, base[b] + np.arange(len(mine)))
            for layer in range(first_layer, first_layer + layers):
                for which in range(2):
                    if hc.layout == 0:
                        cache[dst, layer, which, g] = hc.cache[src, layer, which, g]
                        scale[dst, layer, which, g] = hc.scale[src, layer, which, g]
                    else:
                        cache[layer, which, g, dst] = hc.cache[layer, which, g, src]
                        scale[layer, which, g, dst] = hc.scale[layer, which, g, src]
                if with_weight:
                    weight[layer, g, dst] = hc.weight[layer, g, src]
                    weight[layer, g, hc.rows(b, np.arange(base[b] + len(mine), hc.lens[b]))] = 0
    return cache, scale, weight


def draw_kept(rng, limits, heads, width, dense=False):
    kept = np.full((len(limits), heads, width), -1, dtype=np.int64)
    for b, n in enumerate(limits):
        for g in range(heads):
            m = min(n, width) if dense else int(rng.integers(0, min(n, width) + 1))
            kept[b, g, :m] = np.sort(rng.permutation(n)[:m])
    return kept


@pytest.mark.gpu
@pytest.mark.parametrize("dim,layout,page,layers,first,moved", [
    (128, 0, 0, 1, 0, 1), (64, 0, 0, 3, 1, 2), (128, 3, 0, 2, 0, 2), (64, 3, 48, 1, 0, 1), (128, 0, 16, 2, 1, 1)])
@pytest.mark.parametrize("per_head,with_weight", [(True, True), (True, False), (False, False), (False, True)])
@pytest.mark.parametrize("dense", [False, True])
def test_compact(gpu, pkg, dim, layout, page, layers, first, moved, per_head, with_weight, dense):
    from ppl_nn_b200 import ops
    rng = np.random.default_rng(dim + layout + page + 7 * dense)
    lens = [1, 60, 257, 1500, 3]
    hc = HostCache(rng, lens, 3, dim, layout, page, layers)
    base = np.array([0, 11, 100, 0, 3], dtype=np.int64)
    kept = draw_kept(rng, [n - s for n, s in zip(lens, base)], 3 if per_head else 1, 700, dense)
    want = compact_reference(hc, kept, base, first, moved, with_weight)
    op = ops.KeyValueCacheCompact(ops.KeyValueCacheParam(**hc.param(first)))
    got = [dev(hc.cache), dev(hc.scale), dev(hc.weight)]
    op.forward(dev(kept), dev(hc.starts), dev(base), dev(np.array(lens)), hc.max_len, got[0], got[1],
               weight=got[2] if with_weight else None, num_layers=moved)
    assert op.device_status() == 0
    assert np.array_equal(got[0].cpu().numpy(), want[0])
    assert np.array_equal(got[1].cpu().numpy(), want[1])
    assert np.array_equal(got[2].cpu().numpy(), want[2])


@pytest.mark.gpu
def test_compact_reports_bad_lists(gpu, pkg):
    """Entries out of order or outside their sequence are skipped; nothing outside the sequence is touched."""
    from ppl_nn_b200 import capi, ops
    rng = np.random.default_rng(11)
    hc = HostCache(rng, [50], 1, 64)
    op = ops.KeyValueCacheCompact(ops.KeyValueCacheParam(**hc.param()))
    for bad in ([3, 2, 9, -1], [4, 4, 9, -1], [1, 50, -1, -1], [1, 1 << 40, -1, -1]):
        cache, scale = dev(hc.cache), dev(hc.scale)
        op.forward(dev(np.array([[bad]], dtype=np.int64)), dev(hc.starts), dev(np.array([0])), dev(np.array([50])), 50,
                   cache, scale)
        assert op.device_status() == capi.DEV_KEPT_INVALID, bad
        got = cache.cpu().numpy()
        assert np.array_equal(got[hc.starts[0], 0, 0, 0], hc.cache[hc.starts[0] + bad[0], 0, 0, 0])
        keep = np.ones(hc.max_tokens, dtype=bool)
        keep[hc.starts[0]:hc.starts[0] + 4] = False
        assert np.array_equal(got[keep], hc.cache[keep])


@pytest.mark.gpu
@pytest.mark.parametrize("drop", [1, 3, 64, 200])
@pytest.mark.parametrize("per_head", [True, False])
def test_compact_shifts_by_a_few_rows(gpu, pkg, drop, per_head):
    """Only the first few positions go, so that every row's destination is another row's source: all the segments of a
    list depend on one another."""
    from ppl_nn_b200 import ops
    rng = np.random.default_rng(drop)
    lens = [5000, 4111, 700, 4999, 2048, 201]
    hc = HostCache(rng, lens, 4, 64, 0, 0, 2)
    kept = np.full((len(lens), 4 if per_head else 1, max(lens)), -1, dtype=np.int64)
    for b, n in enumerate(lens):
        for g in range(kept.shape[1]):
            cut = min(drop + (g if per_head else 0), n)
            kept[b, g, :n - cut] = np.arange(cut, n)
    base = np.zeros(len(lens), dtype=np.int64)
    want = compact_reference(hc, kept, base, 0, 2, True)
    op = ops.KeyValueCacheCompact(ops.KeyValueCacheParam(**hc.param()))
    for _ in range(5):
        got = [dev(hc.cache), dev(hc.scale), dev(hc.weight)]
        op.forward(dev(kept), dev(hc.starts), dev(base), dev(np.array(lens)), hc.max_len, *got[:2], weight=got[2],
                   num_layers=2)
        assert op.device_status() == 0
        for g, x in zip(got, want):
            assert np.array_equal(g.cpu().numpy(), x)


# ---- lists that end before their row does --------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("layout,page", [(0, 0), (3, 48)])
@pytest.mark.parametrize("per_head,with_weight", [(True, True), (False, True), (False, False)])
def test_compact_ends_a_list_at_its_first_negative_entry(gpu, pkg, layout, page, per_head, with_weight):
    """What stands behind the terminator -- the list of an earlier step, anything -- is not looked at: neither moved, nor
    reported, nor taken for a part of the list where weights are cleared."""
    from ppl_nn_b200 import ops
    rng = np.random.default_rng(layout + per_head)
    lens = [9, 700, 2000, 300, 64]
    hc = HostCache(rng, lens, 8, 64, layout, page, 2)
    kept = np.sort(rng.integers(0, 2000, size=(len(lens), 8 if per_head else 1, 700)), axis=-1)  # stale: plausible rows
    kept[1] = rng.integers(-3, 1 << 40, size=kept.shape[1:])  # stale: anything, other negative entries too
    for g in range(kept.shape[1]):
        for b, count in enumerate([2, 130 + g, 65, 0, 64]):
            kept[b, g, :count] = np.sort(rng.permutation(lens[b])[:count])
            kept[b, g, count] = -1 - g
    kept[0, 0, :5] = [0, 2, -1, 5, 6]
    want = compact_reference(hc, kept, np.zeros(len(lens), dtype=np.int64), 0, 2, with_weight)
    op = ops.KeyValueCacheCompact(ops.KeyValueCacheParam(**hc.param()))
    for _ in range(3):
        got = [dev(hc.cache), dev(hc.scale), dev(hc.weight)]
        op.forward(dev(kept), dev(hc.starts), dev(np.zeros(len(lens), dtype=np.int64)), dev(np.array(lens)), hc.max_len,
                   got[0], got[1], weight=got[2] if with_weight else None, num_layers=2)
        assert op.device_status() == 0
        for g, x in zip(got, want):
            assert np.array_equal(g.cpu().numpy(), x)


# ---- lists with entries that break the rules -------------------------------------------------------------

def entries_that_move(kept, base, n):
    """(index, position) of a list's entries that count: in range, and above every entry in range before."""
    out, top = [], -1
    for i, p in enumerate(kept):
        if p < 0:
            break
        if i <= p < n - base and p > top:
            out.append((i, p))
            top = p
    return out


def skipping_reference(hc, kept, base, layers):
    cache, scale, weight = hc.cache.copy(), hc.scale.copy(), hc.weight.copy()
    for b in range(len(hc.lens)):
        for g in range(hc.heads):
            mine = kept[b, g if kept.shape[1] > 1 else 0]
            end = int(np.argmax(mine < 0)) if (mine < 0).any() else len(mine)
            pairs = np.array(entries_that_move(mine, base[b], hc.lens[b]), dtype=np.int64).reshape(-1, 2)
            src, dst = hc.rows(b, base[b] + pairs[:, 1]), hc.rows(b, base[b] + pairs[:, 0])
            for layer in range(layers):
                for which in range(2):
                    if hc.layout == 0:
                        cache[dst, layer, which, g] = hc.cache[src, layer, which, g]
                        scale[dst, layer, which, g] = hc.scale[src, layer, which, g]
                    else:
                        cache[layer, which, g, dst] = hc.cache[layer, which, g, src]
                        scale[layer, which, g, dst] = hc.scale[layer, which, g, src]
                weight[layer, g, dst] = hc.weight[layer, g, src]
                weight[layer, g, hc.rows(b, np.arange(base[b] + end, hc.lens[b]))] = 0
    return cache, scale, weight


def spoil(rng, kept, where, kind):
    """Entries that break the rules at the indices `where` of a shifted list."""
    for i in where:
        kept[i] = {"huge": 1 << 40, "low": 0, "same": kept[i - 1] if i else 1 << 33,
                   "over": int(rng.integers(0, len(kept))), "most": np.iinfo(np.int64).max}[kind]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["huge", "low", "same", "over", "most"])
@pytest.mark.parametrize("drop", [1, 70, 200])
@pytest.mark.parametrize("per_head", [True, False])
def test_compact_skips_bad_entries_of_long_lists(gpu, pkg, kind, drop, per_head):
    """Every segment's destinations are others' sources, and entries break the rules at the beginnings, at the ends and in
    the middle of segments: these alone are skipped, and the rows of the others move as they would without them."""
    from ppl_nn_b200 import capi, ops
    rng = np.random.default_rng(drop + per_head)
    lens, base = [3000, 517, 2900, 140], np.array([0, 5, 0, 1], dtype=np.int64)
    hc = HostCache(rng, lens, 8, 64, 0, 0, 2)
    kept = np.full((len(lens), 8 if per_head else 1, max(lens)), -1, dtype=np.int64)
    for b, n in enumerate(lens):
        for g in range(kept.shape[1]):
            count = max(0, n - int(base[b]) - drop)
            kept[b, g, :count] = np.arange(drop, drop + count)
            at = [i for i in (64, 63, 8, 200, 128 + g, 256, 255, 1000, 1024 + g) if i < count]
            spoil(rng, kept[b, g, :count], at, kind)
    want = skipping_reference(hc, kept, base, 2)
    op = ops.KeyValueCacheCompact(ops.KeyValueCacheParam(**hc.param()))
    for _ in range(5):
        got = [dev(hc.cache), dev(hc.scale), dev(hc.weight)]
        op.forward(dev(kept), dev(hc.starts), dev(base), dev(np.array(lens)), hc.max_len, got[0], got[1], weight=got[2],
                   num_layers=2)
        assert op.device_status() == capi.DEV_KEPT_INVALID
        for g, x in zip(got, want):
            assert np.array_equal(g.cpu().numpy(), x)


def wait_range(tops, seg, rows):
    """The earlier segments that the kernel of the moves waits for, as it finds them."""
    below = lambda a, x: int(np.searchsorted(a, x, side="left"))  # noqa: E731
    return below(tops[1:seg + 1], seg * rows), below(tops[:seg], seg * rows + rows - 1) - 1


@pytest.mark.parametrize("rows", [8, 16, 32, 64])
def test_segments_wait_for_all_whose_rows_they_overwrite(rows):
    """The rule by which a segment finds the earlier ones to wait for, on lists with anything in them."""
    rng = np.random.default_rng(rows)
    for trial in range(60):
        n, width = int(rng.integers(1, 900)), int(rng.integers(1, 700))
        kept = np.sort(rng.integers(0, n, size=width)) if trial % 2 else np.arange(width) + int(rng.integers(0, 90))
        bad = rng.random(width) < rng.choice([0, 0.02, 0.3])
        kept = np.where(bad, rng.choice([0, 5, n - 1, n + 3, 1 << 40], size=width), kept)
        moves = entries_that_move(kept, 0, n)
        in_range = np.array([p if i <= p < n else -1 for i, p in enumerate(kept)])
        segments = -(-width // rows)
        tops = np.array([max(in_range[:e * rows], default=-1) for e in range(segments)])
        for seg in range(segments):
            lo, hi = wait_range(tops, seg, rows)
            need = {i // rows for i, p in moves if i // rows < seg and seg * rows <= p < (seg + 1) * rows}
            assert all(lo <= e <= hi for e in need) and hi < seg


@pytest.mark.gpu
@pytest.mark.parametrize("heads,per_head,n", [(8, False, 21001), (2, False, 40100), (1, True, 70100)])  # 8, 32 and 64 rows a segment
@pytest.mark.parametrize("kind", [None, "huge", "over"])
def test_compact_of_lists_with_many_segments(gpu, pkg, heads, per_head, n, kind):
    """More than 1024 segments: the scan of the lists works through them in several steps."""
    from ppl_nn_b200 import capi, ops
    rng = np.random.default_rng(n)
    hc = HostCache(rng, [n, 900], heads, 64)
    base = np.array([3, 0], dtype=np.int64)
    kept = np.full((2, heads if per_head else 1, n), -1, dtype=np.int64)
    for b, m in enumerate(hc.lens):
        count = m - int(base[b]) - 70
        for g in range(kept.shape[1]):
            kept[b, g, :count] = np.arange(70, 70 + count)
            kept[b, g, count + 1:] = 5  # stale
            if kind:
                spoil(rng, kept[b, g, :count], [i for i in (64, 8191, 8192, 16384, 32768, 65536, 65599) if i < count], kind)
    want = skipping_reference(hc, kept, base, 1)
    op = ops.KeyValueCacheCompact(ops.KeyValueCacheParam(**hc.param()))
    for _ in range(3):
        got = [dev(hc.cache), dev(hc.scale), dev(hc.weight)]
        op.forward(dev(kept), dev(hc.starts), dev(base), dev(np.array(hc.lens)), hc.max_len, got[0], got[1], weight=got[2])
        assert op.device_status() == (capi.DEV_KEPT_INVALID if kind else 0)
        for g, x in zip(got, want):
            assert np.array_equal(g.cpu().numpy(), x)
