"""Attention over packed sets (tb_attention) vs the 64-bit form, element by element; the tolerance is
packed_ref.attention_tolerance, half steps of the roundings counted through the formula."""
import math

import pytest
import torch

import packed_ref as ref

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _inputs(seed, nq, nk, h, hk, d, dtype, spread=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    q = (spread * torch.randn((nq, h, d), device="cuda", generator=g)).to(dtype)
    k = torch.randn((nk, hk, d), device="cuda", generator=g).to(dtype)
    v = torch.randn((nk, hk, d), device="cuda", generator=g).to(dtype)
    return q, k, v


def _check(ops, q, k, v, qo, ko, causal=False, scale=None, out_dtype=None, **kw):
    sc = q.shape[2] ** -0.5 if scale is None else scale
    out, lse = ops.attention(q, k, v, ref.table(qo), ref.table(ko), causal=causal, scale=scale, out_dtype=out_dtype,
                             return_lse=True, **kw)
    ops.check_device()
    want, wlse, wgt, reach = ref.attention(q, k, v, qo, ko, causal, sc)
    nk = max([b - a for a, b in zip(ko, ko[1:])] + [1])
    tol = ref.attention_tolerance(want, wgt, reach, q.shape[2], nk, q.dtype, out.dtype)
    assert ref.close(out, want, tol) <= 1.0
    # lse: the score's error, the share that the sum may be off by, and its own rounding
    f = ref.HALF[torch.float32]
    seen = torch.isfinite(wlse)
    e = (q.shape[2] + 3) * f * reach + (64 + nk / 64) * f + 2 ** -13 * (q.dtype != torch.float32) + 4 * f
    assert float(((lse.double() - wlse).abs() - (e + 4 * f * wlse.abs()))[seen].max() if seen.any() else 0.0) <= 0
    none = wlse == -math.inf
    assert bool((lse[none] == -math.inf).all()) and bool((out[none] == 0).all())
    return out


LENGTHS = [
    ([1], [1]),
    ([64], [64]),
    ([129], [127]),
    ([1, 1, 0, 3, 128], [5, 0, 7, 300, 128]),
    ([257, 1, 64, 255], [257, 1, 64, 255]),
    ([300, 20], [1, 513]),
    ([513], [2049]),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("ql,kl", LENGTHS)
def test_lengths(tb, ql, kl, causal, dtype):
    from trellis_cpp_b200 import ops
    q, k, v = _inputs(len(ql) + ql[0], sum(ql), sum(kl), 4, 2, 64, dtype)
    _check(ops, q, k, v, ref.offsets(ql), ref.offsets(kl), causal)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [8, 16, 40, 64, 72, 96, 120, 128])
def test_head_dims(tb, d, dtype):
    from trellis_cpp_b200 import ops
    q, k, v = _inputs(d, 200, 333, 2, 2, d, dtype)
    _check(ops, q, k, v, [0, 90, 200], [0, 133, 333])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("h,hk", [(1, 1), (8, 1), (6, 2), (7, 1), (12, 12), (64, 1), (40, 2)])
def test_grouped_heads(tb, h, hk, causal, dtype):
    from trellis_cpp_b200 import ops
    ql = [37, 1, 150]
    q, k, v = _inputs(h, sum(ql), 400, h, hk, 128, dtype)
    _check(ops, q, k, v, ref.offsets(ql), [0, 37, 200, 400], causal)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("h,hk,d", [(8, 2, 128), (3, 3, 64), (32, 1, 72)])
def test_one_new_token_against_long_caches(tb, h, hk, d, dtype):
    from trellis_cpp_b200 import ops
    kl = [4000, 1, 127, 128, 129, 9000, 640]
    q, k, v = _inputs(h, len(kl), sum(kl), h, hk, d, dtype)
    one = _check(ops, q, k, v, list(range(len(kl) + 1)), ref.offsets(kl), causal=True)
    # causal hides nothing from the last query: the same result to the bit
    assert torch.equal(one, ops.attention(q, k, v, ref.table(list(range(len(kl) + 1))), ref.table(ref.offsets(kl))))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("ql,kl", [([3], [20000]), ([100], [7777]), ([17, 40], [3000, 5001])])
def test_few_queries_many_keys(tb, ql, kl, dtype):
    from trellis_cpp_b200 import ops
    q, k, v = _inputs(7, sum(ql), sum(kl), 2, 1, 128, dtype)
    for causal in (False, True):
        _check(ops, q, k, v, ref.offsets(ql), ref.offsets(kl), causal)


FEW = [      # sets of 16 rows or fewer on average, with heads that share a key head counted as rows
    ([1], [1], 1, 1),
    ([1], [15], 16, 1),
    ([3], [17], 4, 1),
    ([2, 5, 1], [16, 63, 64], 6, 2),
    ([1] * 5, [0, 65, 127, 3, 1000], 8, 2),
    ([16, 16], [40, 700], 2, 2),
    ([0, 0, 40, 0, 1], [9, 0, 500, 70, 2049], 3, 3),      # one set of more rows than a tile
    ([7], [4099], 2, 1),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("d", [8, 40, 64, 72, 128])
@pytest.mark.parametrize("ql,kl,h,hk", FEW)
def test_sets_of_few_rows(tb, ql, kl, h, hk, d, causal, dtype):
    from trellis_cpp_b200 import ops
    q, k, v = _inputs(d + len(ql), sum(ql), sum(kl), h, hk, d, dtype)
    _check(ops, q, k, v, ref.offsets(ql), ref.offsets(kl), causal)


@pytest.mark.parametrize("dtype", DTYPES)
def test_few_rows_strides_and_float32_output(tb, dtype):
    # new tokens as the views of one product, keys and values as the halves of a cache's rows, head-major
    from trellis_cpp_b200 import ops
    h, hk, d, kl = 8, 2, 128, [300, 1, 2000]
    x, _, _ = _inputs(20, 3, 1, h + 2 * hk, 1, d, dtype)
    cache, _, _ = _inputs(21, 2 * hk, 1, sum(kl), 1, d, dtype)
    k, v = cache[:hk].transpose(0, 1), cache[hk:].transpose(0, 1)
    qo, ko = [0, 1, 2, 3], ref.offsets(kl)
    got = _check(ops, x[:, :h], k, v, qo, ko, True)
    wide = _check(ops, x[:, :h], k, v, qo, ko, True, out_dtype=torch.float32)
    assert torch.equal(wide.to(dtype), got)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,start", [(33, 0), (1025, 700), (3001, 40)])
def test_thousands_of_small_sets(tb, n, start, dtype):
    from trellis_cpp_b200 import ops
    g = torch.Generator().manual_seed(n)
    ql = (torch.randint(0, 4, (n,), generator=g) * (torch.rand(n, generator=g) < 0.6)).tolist()
    kl = torch.randint(0, 5, (n,), generator=g).tolist()
    ql[n // 2] = 37
    q, k, v = _inputs(24, sum(ql) + start, sum(kl), 4, 1, 64, dtype)
    _check(ops, q, k, v, ref.offsets(ql, start), ref.offsets(kl), True)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("qo,ko", [([0, 3, 2, 6], [0, 50, 90, 128]), ([-1, 2, 4, 6], [0, 50, 90, 128]),
                                   ([0, 2, 4, 6], [0, 90, 50, 128]), ([0, 2, 4, 6], [0, 50, 90, 129]),
                                   ([0, 0, 0, 6], [0, 50, 40, 128])])
def test_few_rows_bad_tables_are_reported(tb, qo, ko, dtype):
    from trellis_cpp_b200 import ops
    q, k, v = _inputs(25, 6, 128, 2, 2, 64, dtype)
    ops.attention(q, k, v, ref.table(qo), ref.table(ko))
    with pytest.raises(ops.TBError) as e:
        ops.check_device()
    assert e.value.status == 5 and "offset table" in str(e.value)
    _check(ops, q, k, v, [0, 2, 6], [0, 50, 128])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("scale,spread", [(1e-4, 1.0), (0.125, 20.0), (2.0, 3.0)])
def test_few_rows_flat_steep_and_rising_scores(tb, scale, spread, dtype):
    from trellis_cpp_b200 import ops
    q, k, v = _inputs(22, 4, 3000, 2, 2, 64, dtype, spread)
    _check(ops, q, k, v, [0, 1, 4], [0, 900, 3000], True, scale=scale)
    k = (k.abs() * torch.linspace(0.1, 4, 3000, device="cuda")[:, None, None]).to(dtype)
    _check(ops, q.abs(), k, v, [0, 1, 4], [0, 900, 3000], False, scale=scale)


@pytest.mark.parametrize("dtype", DTYPES)
def test_few_rows_where_the_next_set_holds_no_numbers(tb, dtype):
    from trellis_cpp_b200 import ops
    q, k, v = _inputs(23, 2, 2000, 4, 1, 128, dtype)
    k[1003:] = math.nan
    v[1003:] = math.inf
    out = ops.attention(q, k, v, ref.table([0, 1, 2]), ref.table([0, 1003, 2000]))
    want, _, wgt, reach = ref.attention(q[:1], k[:1003], v[:1003], [0, 1], [0, 1003], False, 128 ** -0.5)
    tol = ref.attention_tolerance(want, wgt, reach, 128, 1003, dtype, dtype)
    assert ref.close(out[:1], want, tol) <= 1.0
    assert bool(torch.isnan(out[1:]).all())
    k[1003:] = 0
    k[5, 0, 3] = math.nan                          # in the first range of the keys, then in the last
    assert bool(torch.isnan(ops.attention(q[:1], k[:1003], v[:1003])).all())
    k[5] = 0
    k[1002] = math.nan
    assert bool(torch.isnan(ops.attention(q[:1], k[:1003], v[:1003])).all())
    ops.check_device()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_many_sets(tb, dtype):
    from trellis_cpp_b200 import ops
    g = torch.Generator().manual_seed(1)
    ql = torch.randint(0, 20, (700,), generator=g).tolist()
    kl = torch.randint(0, 30, (700,), generator=g).tolist()
    q, k, v = _inputs(2, sum(ql), sum(kl), 4, 4, 64, dtype)
    _check(ops, q, k, v, ref.offsets(ql), ref.offsets(kl), True)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("scale,spread", [(1e-4, 1.0), (0.125, 20.0), (2.0, 3.0)])
def test_flat_and_steep_scores(tb, scale, spread, dtype):
    from trellis_cpp_b200 import ops
    q, k, v = _inputs(11, 150, 700, 2, 2, 64, dtype, spread)
    _check(ops, q, k, v, [0, 150], [0, 700], True, scale=scale)


@pytest.mark.parametrize("dtype", DTYPES)
def test_rising_maximum(tb, dtype):
    # each block of keys scores higher than the one before: the running maximum moves every time
    from trellis_cpp_b200 import ops
    q, k, v = _inputs(12, 140, 1200, 1, 1, 64, dtype)
    q = q.abs()
    k = (k.abs() * torch.linspace(0.1, 4, 1200, device="cuda")[:, None, None]).to(dtype)
    _check(ops, q, k, v, [0, 140], [0, 1200])
    _check(ops, q, k.flip(0).contiguous(), v, [0, 140], [0, 1200])


@pytest.mark.parametrize("dtype", DTYPES)
def test_views_of_one_product(tb, dtype):
    from trellis_cpp_b200 import ops
    h, hk, d, n = 6, 2, 64, 301
    x, _, _ = _inputs(3, n, 1, h + 2 * hk, 1, d, dtype)
    qo = [0, 100, 301]
    _check(ops, x[:, :h], x[:, h:h + hk], x[:, h + hk:], qo, qo, True)


@pytest.mark.parametrize("dtype", DTYPES)
def test_head_major_strides_and_given_out(tb, dtype):
    from trellis_cpp_b200 import ops
    q, k, v = _inputs(4, 130, 260, 4, 2, 64, dtype)
    hm = lambda t: t.transpose(0, 1).contiguous().transpose(0, 1)  # noqa: E731  [heads][rows][dim] memory
    want = _check(ops, q, k, v, [0, 130], [0, 260])
    out = torch.full((4, 140, 64), 7.0, dtype=dtype, device="cuda").transpose(0, 1)
    got = ops.attention(hm(q), hm(k), hm(v), out=out[5:135])
    assert got.data_ptr() == out[5:135].data_ptr() and torch.equal(got, want)
    assert bool((out[:5] == 7).all()) and bool((out[135:] == 7).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("ql,kl", [([50, 0, 131], [100, 3, 260]), ([1, 1, 1], [300, 0, 1000])])
def test_rows_outside_the_sets(tb, ql, kl, causal, dtype):
    """Rows before, between (there are none) and behind the sets: keys and values there hold no numbers and
    have no effect; output rows there keep their values."""
    from trellis_cpp_b200 import ops
    qo, ko = ref.offsets(ql, 9), ref.offsets(kl, 13)
    q, k, v = _inputs(5, qo[-1] + 140, ko[-1] + 150, 4, 4, 64, dtype)
    for bad in (math.nan, math.inf, -math.inf):
        for t, o in ((k, ko), (v, ko), (q, qo)):
            t[:o[0]] = bad
            t[o[-1]:] = bad
        out = torch.full(q.shape, 5.0, dtype=dtype, device="cuda")
        lse = _check(ops, q, k, v, qo, ko, causal, out=out)
        assert lse.data_ptr() == out.data_ptr()
        assert bool((out[:qo[0]] == 5).all()) and bool((out[qo[-1]:] == 5).all())
        assert bool(torch.isfinite(out).all())


@pytest.mark.parametrize("dtype", DTYPES)
def test_next_set_holds_no_numbers(tb, dtype):
    # keys and values of one set (the rows right behind another's last key) hold no numbers
    from trellis_cpp_b200 import ops
    q, k, v = _inputs(6, 60, 190, 2, 2, 64, dtype)
    k[70:] = math.nan
    v[70:] = math.inf
    out = ops.attention(q, k, v, ref.table([0, 40, 60]), ref.table([0, 70, 190]))
    want, _, wgt, reach = ref.attention(q[:40], k[:70], v[:70], [0, 40], [0, 70], False, 64 ** -0.5)
    tol = ref.attention_tolerance(want, wgt, reach, 64, 70, dtype, dtype)
    assert ref.close(out[:40], want, tol) <= 1.0
    assert bool(torch.isnan(out[40:]).all())       # a score that is no number makes its rows none


@pytest.mark.parametrize("dtype", DTYPES)
def test_values_that_are_no_numbers_reach_their_rows(tb, dtype):
    from trellis_cpp_b200 import ops
    q, k, v = _inputs(8, 40, 300, 2, 2, 64, dtype)
    v[170, 0, 3] = math.nan
    k[33, 1] = math.nan
    out = ops.attention(q, k, v)
    assert bool(torch.isnan(out[:, 0, 3]).all()) and bool(torch.isnan(out[:, 1]).all())
    keep = [i for i in range(64) if i != 3]
    assert bool(torch.isfinite(out[:, 0, keep]).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_float32_output(tb, dtype):
    from trellis_cpp_b200 import ops
    q, k, v = _inputs(9, 200, 300, 4, 2, 128, dtype)
    out = _check(ops, q, k, v, [0, 200], [0, 300], out_dtype=torch.float32)
    assert out.dtype == torch.float32
    assert torch.equal(out.to(dtype), ops.attention(q, k, v))


@pytest.mark.parametrize("dtype", DTYPES)
def test_repeats_to_the_bit(tb, dtype):
    from trellis_cpp_b200 import ops
    q, k, v = _inputs(10, 300, 5000, 4, 2, 128, dtype)
    a = ops.attention(q, k, v)
    b = ops.attention(q[:3], k, v)
    for _ in range(3):
        assert torch.equal(a, ops.attention(q, k, v)) and torch.equal(b, ops.attention(q[:3], k, v))


@pytest.mark.parametrize("dtype", DTYPES)
def test_nothing_to_do(tb, dtype):
    from trellis_cpp_b200 import ops
    q, k, v = _inputs(1, 5, 7, 2, 2, 64, dtype)
    assert ops.attention(q[:0], k, v).shape == (0, 2, 64)
    out, lse = ops.attention(q, k[:0], v[:0], return_lse=True)      # no keys at all
    assert bool((out == 0).all()) and bool((lse == -math.inf).all())
    assert ops.attention(q, k, v, ref.table([0]), ref.table([0])).shape == q.shape   # no sets
    ops.check_device()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("nq,nk", [(300, 300), (2, 6000)])
def test_captured_call_follows_its_tables(tb, nq, nk, dtype):
    # two graphs and an eager call, each with workspace of its own, replayed at the same time
    from trellis_cpp_b200 import ops
    q, k, v = _inputs(13, nq, nk, 4, 2, 128, dtype)
    qo, ko = ref.table([0, nq // 2, nq]), ref.table([0, nk // 3, nk])
    ops.attention(q, k, v, qo, ko)
    graphs, outs, streams = [], [], [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for i in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(ops.attention(q, k, v, qo, ko, causal=i == 1))
        graphs.append(gr)
    qo.copy_(ref.table([0, 1, nq - 1]))
    ko.copy_(ref.table([5, nk // 2, nk - 1]))
    torch.cuda.synchronize()
    for _ in range(3):
        for gr, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                gr.replay()
        eager = ops.attention(q, k, v, qo, ko)
    torch.cuda.synchronize()
    ops.check_device()
    assert torch.equal(outs[0][:nq - 1], eager[:nq - 1])
    assert torch.equal(outs[1][:nq - 1], ops.attention(q, k, v, qo, ko, causal=True)[:nq - 1])
    want, _, wgt, reach = ref.attention(q, k, v, [0, 1, nq - 1], [5, nk // 2, nk - 1], False, 128 ** -0.5)
    tol = ref.attention_tolerance(want, wgt, reach, 128, nk, dtype, dtype)
    assert ref.close(eager, want, tol) <= 1.0


@pytest.mark.parametrize("dtype", DTYPES)
def test_calls_on_two_streams(tb, dtype):
    from trellis_cpp_b200 import ops
    q, k, v = _inputs(14, 500, 4000, 4, 2, 64, dtype)
    want, few = ops.attention(q, k, v), ops.attention(q[:2], k, v)
    torch.cuda.synchronize()
    got = []
    for i in range(6):
        with torch.cuda.stream(torch.cuda.Stream()):
            got.append((ops.attention(q, k, v), ops.attention(q[:2], k, v)))
    torch.cuda.synchronize()
    for a, b in got:
        assert torch.equal(a, want) and torch.equal(b, few)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_far_apart(tb, dtype):
    # element offsets past 2^31: rows of a wide cache
    from trellis_cpp_b200 import ops
    wide = 1 << 23
    nk = 400 if dtype == torch.bfloat16 else 300
    store = torch.empty((nk, wide), dtype=dtype, device="cuda")
    q, k, v = _inputs(15, 20, nk, 2, 1, 64, dtype)
    kk, vv = store[:, wide - 128:wide - 64].unsqueeze(1), store[:, 64:128].unsqueeze(1)
    kk.copy_(k)
    vv.copy_(v)
    assert torch.equal(ops.attention(q, kk, vv), ops.attention(q, k, v))
    assert torch.equal(ops.attention(q[:5], kk, vv), ops.attention(q[:5], k, v))
    ops.check_device()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("qo,ko", [([0, 30, 20, 64], [0, 50, 90, 128]), ([0, 20, 40, 100], [0, 50, 90, 128]),
                                   ([-5, 20, 40, 64], [0, 50, 90, 400]), ([0, 20, 40, 64], [0, 90, 50, 128])])
def test_bad_tables_are_reported(tb, qo, ko, dtype):
    from trellis_cpp_b200 import ops
    q, k, v = _inputs(16, 64, 128, 2, 2, 64, dtype)
    ops.attention(q, k, v, ref.table(qo), ref.table(ko))
    with pytest.raises(ops.TBError) as e:
        ops.check_device()
    assert e.value.status == 5 and "offset table" in str(e.value)
    _check(ops, q, k, v, [0, 20, 64], [0, 50, 128])          # the next call is sound


def test_refusals(tb):
    from trellis_cpp_b200 import ops
    q, k, v = _inputs(17, 10, 20, 4, 2, 64, torch.bfloat16)
    o2, o3 = ref.table([0, 10]), ref.table([0, 5, 10])
    for call, kind in [
        (lambda: ops.attention(q.cpu(), k, v), ValueError),
        (lambda: ops.attention(q, k.float(), v), ValueError),
        (lambda: ops.attention(q, k, v[:10]), ValueError),
        (lambda: ops.attention(q[..., ::2], k[..., ::2], v[..., ::2]), ValueError),
        (lambda: ops.attention(q, k, v, None, o2), ValueError),
        (lambda: ops.attention(q, k, v, o2, o3), ValueError),
        (lambda: ops.attention(q, k, v, o2.long(), o2), ValueError),
        (lambda: ops.attention(q, k, v, out=torch.empty_like(q)[:5]), ValueError),
        (lambda: ops.attention(q[:, :3], k, v), ops.TBError),                       # 3 heads on 2 key heads
        (lambda: ops.attention(q, k, v, scale=0.0), ops.TBError),
        (lambda: ops.attention(q, k, v, scale=-1.0), ops.TBError),
        (lambda: ops.attention(q, k, v, scale=math.nan), ops.TBError),
        (lambda: ops.attention(q[..., :60], k[..., :60], v[..., :60]), ops.TBError),    # head_dim % 8
        (lambda: ops.attention(q, k, v, out_dtype=torch.float16), ops.TBError),
        (lambda: ops.attention(q, k, v, out=q), ops.TBError),
        (lambda: ops.attention(q.expand(10, 4, 64), k[:1].expand(20, 2, 64), v), ops.TBError),   # rows 0 apart
        (lambda: ops.attention(torch.zeros((10, 4, 136), dtype=q.dtype, device="cuda"),
                               torch.zeros((20, 2, 136), dtype=q.dtype, device="cuda"),
                               torch.zeros((20, 2, 136), dtype=q.dtype, device="cuda")), ops.TBError),
        (lambda: ops.attention(torch.zeros((10, 4, 68), dtype=q.dtype, device="cuda")[..., 4:], k, v), ops.TBError),
    ]:
        with pytest.raises(kind):
            call()
    ops.check_device()
