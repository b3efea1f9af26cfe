"""Attention of drafted token trees over the INT8 cache, against plain numpy in 64 bits."""
import ctypes
import math

import numpy as np
import pytest

from test_cache_ops import FAKE, HostCache, _params, dev, gpu, starts_of  # noqa: F401  (gpu is a fixture)


def _tree_call(lib, p, q=FAKE, parents=FAKE, seq=FAKE, cache=FAKE, scale=FAKE, out=FAKE, ws=FAKE, n=1 << 40):
    return lib.tree_attn_forward(p, q, parents, seq, FAKE, FAKE, cache, scale, out, ws, n, None)


@pytest.mark.parametrize("field,value,expect", [
    ("quant_group", 16, "RC_UNSUPPORTED"), ("head_dim", 96, "RC_UNSUPPORTED"), ("num_kv_heads", 5, "RC_INVALID_VALUE"),
    ("max_seqlen", 1025, "RC_UNSUPPORTED"), ("max_kvlen", 1 << 31, "RC_UNSUPPORTED"), ("batch", 65536, "RC_UNSUPPORTED"),
])
def test_attributes_are_refused(built_lib, pkg, field, value, expect):
    from ppl_nn_b200 import capi
    p = _params(built_lib, capi)
    setattr(p, field, value)
    assert built_lib.status_str(_tree_call(built_lib, p)) == expect
    rc, _ = built_lib.tree_attn_workspace_size(p)
    assert built_lib.status_str(rc) == expect


@pytest.mark.parametrize("kw,expect", [
    (dict(scale=None), "RC_UNSUPPORTED"), (dict(q=None), "RC_NOT_FOUND"), (dict(out=None), "RC_NOT_FOUND"),
    (dict(out=ctypes.c_void_p(4096 + 16)), "RC_INVALID_VALUE"), (dict(q=ctypes.c_void_p(4104)), "RC_INVALID_VALUE"),
    (dict(parents=ctypes.c_void_p(4100)), "RC_INVALID_VALUE"),
])
def test_arguments_are_refused(built_lib, pkg, kw, expect):
    import torch
    from ppl_nn_b200 import capi
    p = _params(built_lib, capi)
    assert built_lib.status_str(_tree_call(built_lib, p, **kw)) == expect
    if not torch.cuda.is_available():
        assert built_lib.status_str(_tree_call(built_lib, p, parents=None)) == "RC_NO_DEVICE_CODE"
    assert _tree_call(built_lib, _params(built_lib, capi, batch=0, total_tokens=0), q=None, out=None) == capi.SUCCESS


def test_more_blocks_than_32_bits_count_are_refused(built_lib, pkg):
    """Blocks of a (sequence, kv head): 64 positions x 128 query rows."""
    from ppl_nn_b200 import capi
    for heads, max_seqlen, max_kvlen, expect in (
            (4096, 1024, 1 << 23, "RC_UNSUPPORTED"),  # 2^15 x 2^17
            (4096, 1024, (1 << 22) - 64, "RC_SUCCESS"), (8, 1024, 0x7fff0000, "RC_SUCCESS")):
        p = _params(built_lib, capi, num_heads=heads, num_kv_heads=1, max_seqlen=max_seqlen, max_kvlen=max_kvlen)
        rc, _ = built_lib.tree_attn_workspace_size(p)
        assert built_lib.status_str(rc) == expect
        if expect != "RC_SUCCESS":
            assert built_lib.status_str(_tree_call(built_lib, p)) == expect


def draw_parents(rng, n, kind):
    if kind == "chain":
        return list(range(-1, n - 1))
    if kind == "roots":
        return [-1] * n
    if kind == "star":
        return [-1] + [0] * (n - 1)
    return [-1 if i == 0 else int(rng.integers(-1, i)) for i in range(n)]


def tree_reference(hc, q, parents, start, n, heads, layer):
    """Output, and how far a result may be off each value, in 64 bits.

    Keys, weights, values and the output are each rounded to fp16, by at most u = 2^-11 of the value.  The rounding
    errors of a score's products are independent and bounded by u |q k|: their sum exceeds 6 times the root of the sum
    of the squared bounds with a probability below 2 exp(-18).  A score's error enters a weight once by itself and
    once by the normaliser; rounding a weight and a value adds u each, and 2^-16 covers the exponentials and the fp32
    sums.  Weights below fp16's normal range are off by 2^-25 of the largest, in the numerator and in the sum."""
    group, u = heads // hc.heads, 2.0 ** -11
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    first = 0
    for b in range(len(hc.lens)):
        rows = hc.rows(b, np.arange(start[b] + n[b]))
        for g in range(hc.heads):
            k, v = hc.values(0, layer, g, rows), hc.values(1, layer, g, rows)
            for i in range(n[b]):
                see = list(range(start[b]))
                a = i
                while a >= 0:
                    see.append(start[b] + a)
                    a = parents[first + a]
                for h in range(group):
                    x = q[first + i, g * group + h].astype(np.float64)
                    s = k[see] @ x / math.sqrt(hc.dim)
                    p = np.exp(s - s.max())
                    p /= p.sum()
                    off = 6 * u * np.sqrt((k[see] ** 2) @ (x ** 2)).max() / math.sqrt(hc.dim)
                    o = p @ v[see]
                    mag = p @ np.abs(v[see])
                    out[first + i, g * group + h] = o
                    tol[first + i, g * group + h] = (mag * (2 * off + 2 * u + 2.0 ** -16) + u * np.abs(o)
                                                     + 2 * len(see) * 2.0 ** -25 * np.abs(v[see]).max())
        first += n[b]
    return out, tol


TREE_CASES = [
    # heads, kv heads, dim, start, n, kind, layout, page, layers, layer
    (8, 8, 64, [10, 57, 123, 248], [7, 5, 3, 1], "tree", 0, 0, 1, 0),
    (8, 2, 128, [0, 1, 63, 64, 65], [1, 2, 1, 5, 64], "tree", 0, 0, 1, 0),
    (4, 1, 128, [5000], [13], "tree", 0, 0, 1, 0),
    (16, 2, 64, [0, 300], [65, 0], "tree", 3, 0, 2, 1),
    (8, 2, 128, [100, 0, 700], [33, 16, 31], "roots", 0, 16, 1, 0),
    (8, 1, 128, [40, 1000], [70, 9], "tree", 3, 48, 3, 1),
    (6, 2, 64, [77], [130], "chain", 0, 128, 1, 0),
    (3, 1, 128, [513, 64], [1, 1], "tree", 0, 0, 2, 1),
    (8, 4, 128, [250, 2040], [60, 19], "star", 3, 128, 1, 0),
    (32, 8, 128, [129, 64, 30, 1], [4, 8, 12, 16], "tree", 0, 0, 1, 0),
]


def run_tree(hc, q, parents, start, n, heads, layer, **kw):
    from ppl_nn_b200 import ops
    op = ops.TreeAttention(ops.MultiHeadCacheAttentionParam(num_heads=heads, num_kv_heads=hc.heads, head_dim=hc.dim,
                                                            **hc.param(layer)))
    out = op.forward(dev(q), None if parents is None else dev(np.array(parents, dtype=np.int64)), dev(starts_of(n)),
                     dev(hc.starts), dev(np.array(start, dtype=np.int64)), kw.get("max_n", max(n)),
                     kw.get("max_len", hc.max_len), dev(hc.cache), dev(hc.scale))
    return out.cpu().numpy().astype(np.float64), op.device_status()


@pytest.mark.gpu
@pytest.mark.parametrize("case", TREE_CASES, ids=str)
def test_tree_attention(gpu, pkg, case):  # noqa: F811
    heads, kv_heads, dim, start, n, kind, layout, page, layers, layer = case
    rng = np.random.default_rng(len(str(case)))
    hc = HostCache(rng, [s + m for s, m in zip(start, n)], kv_heads, dim, layout, page, layers)
    q = rng.standard_normal((sum(n), heads, dim)).astype(np.float16)
    parents = sum([draw_parents(rng, m, kind) for m in n], [])
    want, tol = tree_reference(hc, q, parents, start, n, heads, layer)
    got, status = run_tree(hc, q, parents, start, n, heads, layer)
    assert status == 0
    assert np.all(np.abs(got - want) <= tol), float((np.abs(got - want) / tol).max())
    if kind == "chain":  # without parents: the same chain
        same, status = run_tree(hc, q, None, start, n, heads, layer)
        assert status == 0 and np.array_equal(same, got)
    # longer bounds than needed change the split of the work, not what is computed
    wide, status = run_tree(hc, q, parents, start, n, heads, layer, max_n=max(n) + 70, max_len=hc.max_len + (0 if page else 900))
    assert status == 0 and np.all(np.abs(wide - want) <= tol)


@pytest.mark.gpu
def test_tree_of_one_token_is_a_decode_step(gpu, pkg):  # noqa: F811
    """One drafted token per sequence, already in the cache: the decode operator's result."""
    from ppl_nn_b200 import capi, ops
    rng = np.random.default_rng(2)
    start, n = [0, 40, 1999], [1, 1, 1]
    hc = HostCache(rng, [s + 1 for s in start], 2, 128)
    q = rng.standard_normal((3, 8, 128)).astype(np.float16)
    got, status = run_tree(hc, q, [-1, -1, -1], start, n, 8, 0)
    assert status == 0
    op = ops.MultiHeadCacheAttention(ops.MultiHeadCacheAttentionParam(num_heads=8, num_kv_heads=2, head_dim=128,
                                                                      **hc.param()))
    kv = dev(np.zeros((3, 2, 128), dtype=np.float16))
    ref = op.forward(dev(q), kv, kv, dev(starts_of(n)), dev(starts_of(hc.lens)), dev(hc.starts),
                     dev(np.array(start, dtype=np.int64)), 3, 1, 2000, dev(hc.cache), dev(hc.scale),
                     phase_mask=capi.PHASE_DECODE).cpu().numpy().astype(np.float64)
    _, tol = tree_reference(hc, q, [-1] * 3, start, n, 8, 0)
    assert np.all(np.abs(got - ref) <= 2 * tol)


@pytest.mark.gpu
def test_tree_attention_reports_bad_inputs(gpu, pkg):  # noqa: F811
    """A parent that does not come before its child counts as -1; a cut length and a row outside the cache are
    reported; what is behind the sequences does not matter."""
    from ppl_nn_b200 import capi
    rng = np.random.default_rng(4)
    start, n = [20, 90], [5, 6]
    hc = HostCache(rng, [25, 96], 2, 64)
    for b in range(2):
        hc.scale[hc.starts[b] + hc.lens[b]:(hc.starts[b + 1] if b == 0 else None)] = np.nan
    q = rng.standard_normal((11, 4, 64)).astype(np.float16)
    good = [-1, 0, -1, 2, 3, -1, 0, 1, 2, -1, 4]
    bad = [-7, 0, 9, 2, 3, 0, 0, 1, 2, 4, 4]  # differs where a parent is not before its child: those are roots
    want, tol = tree_reference(hc, q, good, start, n, 4, 0)
    got, status = run_tree(hc, q, bad, start, n, 4, 0)
    assert status == capi.DEV_PARENT_INVALID
    assert np.all(np.abs(got - want) <= tol)
    _, status = run_tree(hc, q, good, start, n, 4, 0, max_len=60)
    assert status == capi.DEV_LENGTH_CLAMPED
    hc.starts[1] = hc.max_tokens - 40
    got, status = run_tree(hc, q, good, start, n, 4, 0)
    assert status & capi.DEV_ROW_OUT_OF_RANGE
    assert np.all(np.abs(got[:5] - want[:5]) <= tol[:5])


@pytest.mark.gpu
@pytest.mark.parametrize("above", [14.0, 17.0, 18.0, 19.0])
def test_what_stands_behind_a_dominant_token_is_kept(gpu, pkg, above):  # noqa: F811
    """131071 positions whose scores spread by 1 around a mean, and a first token (a sink) that stands `above` over it, with
    values near zero: the others hold 10 to 0.1 % of the weight and nearly all of the output.  All the sequences read the
    same rows, so that most of them are worked on from the sink to the end by one CTA.

    Tolerance: a score is a sum of 2 Dh exact products in fp32 (Dh / 8 instructions, 2^-22 of the products' magnitudes
    each), an error of the exponent of a weight and of the normaliser; weights, values and the output are rounded to
    fp16 (2^-11); fp16 holds a weight as 2^7 or more times its ratio to the row's largest, so that below the normal range
    the rounding, at most 2^-25, is 2^-32 of the largest, in the numerator and in the sum; 2^-16 covers the exponentials
    and the fp32 sums."""
    import torch
    from ppl_nn_b200 import ops
    rng = np.random.default_rng(int(above))
    heads, dim, hist, batch, u = 2, 64, 131071, 300, 2.0 ** -11
    hc = HostCache(rng, [hist + 1], 1, dim)
    rows = hc.rows(0, np.arange(hist + 1))
    sign = rng.choice([-1, 1], size=(heads, dim))
    q = np.broadcast_to(sign, (batch, heads, dim)).astype(np.float16)
    # uniform codes have a spread of 73.3: 8 * 73.3 * scale / 8 = 1
    hc.scale[rows, 0, 0] = np.float16(1 / 73.3)
    hc.cache[rows[0], 0, 0, 0] = np.where(sign[0] == sign[1], 127, 0) * sign[0]  # both heads' sink
    agree = int((sign[0] == sign[1]).sum())
    hc.scale[rows[0], 0, 0] = np.float16(above * 8 / (127 * agree))
    hc.cache[rows, 0, 1] = rng.integers(30, 128, size=(hist + 1, 1, dim))  # values of one sign: nothing cancels
    hc.scale[rows[0], 0, 1] = np.float16(1e-5)
    k, v = hc.values(0, 0, 0, rows), hc.values(1, 0, 0, rows)
    s = (k @ sign.T.astype(np.float64)) / math.sqrt(dim)  # [positions, heads]
    p = np.exp(s - s.max(0))
    p /= p.sum(0)
    want, mag = p.T @ v, p.T @ np.abs(v)
    off = (dim / 8) * 2.0 ** -22 * np.abs(k).sum(1).max() / math.sqrt(dim)
    tol = mag * (2 * off + 2 * u + 2.0 ** -16) + u * np.abs(want) + 2 * len(rows) * 2.0 ** -32 * np.abs(v).max()
    op = ops.TreeAttention(ops.MultiHeadCacheAttentionParam(num_heads=heads, num_kv_heads=1, head_dim=dim, **hc.param()))
    i64 = lambda x: torch.tensor(x, dtype=torch.int64, device=gpu)  # noqa: E731
    out = op.forward(dev(q), None, torch.arange(batch + 1, device=gpu), i64([int(hc.starts[0])] * batch), i64([hist] * batch), 1,
                     hist + 1, dev(hc.cache), dev(hc.scale))
    assert op.device_status() == 0
    got = out.cpu().numpy().astype(np.float64)
    assert np.all(np.abs(got - want) <= tol), float((np.abs(got - want) / tol).max())


@pytest.mark.gpu
@pytest.mark.parametrize("shift", [0, 1, 6, -1, -6])
def test_an_output_over_the_query_is_refused(gpu, pkg, shift):  # noqa: F811
    """Other parts of the call still read what this one would write, also where the two only overlap."""
    import torch
    from ppl_nn_b200 import ops
    hc = HostCache(np.random.default_rng(0), [30], 2, 64)
    room = torch.zeros(21, 4, 64, dtype=torch.float16, device=gpu)
    op = ops.TreeAttention(ops.MultiHeadCacheAttentionParam(num_heads=4, num_kv_heads=2, head_dim=64, **hc.param()))
    i64 = lambda x: torch.tensor(x, dtype=torch.int64, device=gpu)  # noqa: E731
    args = (None, i64([0, 7]), dev(hc.starts), i64([20]), 7, 30, dev(hc.cache), dev(hc.scale))
    with pytest.raises(ops.OpError):
        op.forward(room[7:14], *args, attn_output=room[7 + shift:14 + shift])
    for beside in (0, 14):
        op.forward(room[7:14], *args, attn_output=room[beside:beside + 7])
        assert op.device_status() == 0
