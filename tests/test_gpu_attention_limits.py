"""Attention (tb_attention) at the ends of what scores and lengths may be: rows whose scores are all
-inf, in calls whose keys are cut into ranges and in others; rows of hundreds of thousands to hundreds
of millions of keys. The tolerance is that of packed_ref.attention_tolerance where nothing else is said."""
import math

import pytest
import torch

import packed_ref as ref

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 72, 128])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("ql,kl", [([1, 1, 1], [40, 9, 40]), ([1, 1, 1], [9000, 300, 4000]), ([200, 40, 3], [130, 260, 700]),
                                   ([200, 1, 30], [9000, 40, 6000]), ([2500, 600, 900], [900, 130, 257])])
def test_scores_that_are_all_minus_infinity(tb, ql, kl, causal, dtype, d):
    """Set 0: every score -inf. Set 1: none. Set 2: those of its first half, which causal may leave a row
    alone with."""
    from trellis_cpp_b200 import ops
    qo, ko = ref.offsets(ql), ref.offsets(kl)
    h = 12 if ql[0] == 2500 else 2
    g = torch.Generator(device="cuda").manual_seed(d + ql[0])
    q = torch.randn((qo[-1], h, d), device="cuda", generator=g).to(dtype)
    k = torch.randn((ko[-1], h, d), device="cuda", generator=g).to(dtype)
    v = torch.randn((ko[-1], h, d), device="cuda", generator=g).to(dtype)
    q[..., 0] = 1.0
    finite = k.clone()
    k[:kl[0], :, 0] = -math.inf
    k[ko[2]:ko[2] + kl[2] // 2, :, 0] = -math.inf
    out, lse = ops.attention(q, k, v, ref.table(qo), ref.table(ko), causal=causal, return_lse=True)
    ops.check_device()
    want, wlse, wgt, _ = ref.attention(q, k, v, qo, ko, causal, d ** -0.5)
    _, _, _, reach = ref.attention(q, finite, v, qo, ko, causal, d ** -0.5)      # of the scores that are numbers
    tol = ref.attention_tolerance(want, wgt, reach, d, max(kl), dtype, dtype)
    assert ref.close(out, want, tol) <= 1.0
    none = wlse == -math.inf
    assert bool(none[:ql[0]].all())
    assert bool((lse == -math.inf)[none].all()) and bool((out[none] == 0).all()) and bool(torch.isfinite(lse[~none]).all())


def _sampled(ops, q, k, v, qo, ko, rows, causal=False, **kw):
    """The call against the 64-bit form at some rows: (set, row of the set)."""
    out, lse = ops.attention(q, k, v, ref.table(qo), ref.table(ko), causal=causal, return_lse=True, **kw)
    ops.check_device()
    d, f = q.shape[2], ref.HALF[torch.float32]
    for s, t in rows:
        n, a, b = qo[s + 1] - qo[s], ko[s], ko[s + 1]
        end = max(a, b - (n - 1 - t)) if causal else b
        i = qo[s] + t
        want, wlse, wgt, reach = ref.attention(q[i:i + 1], k[a:end], v[a:end], [0, 1], [0, end - a], False, d ** -0.5)
        tol = ref.attention_tolerance(want, wgt, reach, d, end - a, q.dtype, out.dtype)
        assert ref.close(out[i:i + 1], want, tol) <= 1.0, (s, t)
        e = (d + 3) * f * reach + (64 + (end - a) / 64) * f + 2 ** -13 + 4 * f * (1 + wlse.abs())
        assert bool(((lse[i:i + 1].double() - wlse).abs() <= e).all() or end == a), (s, t)
    return out


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("order", ["flat", "rising", "falling"])
@pytest.mark.parametrize("ql,kl,h,d", [
    ([5120], [100003], 4, 64), ([5120], [100003], 4, 128), ([5120], [98304], 4, 72),     # one range of keys
    ([100] + [3] * 160, [70001] + [40] * 160, 1, 128), ([20] * 170, [70001] + [300] * 169, 1, 40),
    ([1280], [600000], 4, 64), ([300, 5], [700001, 9], 8, 128),                          # several, each a long one
])
def test_ranges_of_more_keys_than_one_accumulation_takes(tb, ql, kl, h, d, order, dtype):
    from trellis_cpp_b200 import ops
    qo, ko = ref.offsets(ql), ref.offsets(kl)
    g = torch.Generator(device="cuda").manual_seed(d + ql[0])
    q = torch.randn((qo[-1], h, d), device="cuda", generator=g).to(dtype)
    k = torch.randn((ko[-1], h, d), device="cuda", generator=g)
    v = torch.randn((ko[-1], h, d), device="cuda", generator=g).to(dtype)
    if order != "flat":
        q = q.abs()
        ramp = torch.linspace(0.1, 3, ko[-1], device="cuda")[:, None, None]
        k = k.abs() * (ramp if order == "rising" else ramp.flip(0))
    k = k.to(dtype)
    rows = [(0, 0), (0, ql[0] // 2), (0, ql[0] - 1)] + [(len(ql) - 1, t) for t in (0, ql[-1] - 1) if len(ql) > 1]
    _sampled(ops, q, k, v, qo, ko, rows)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [64, 128])
def test_causal_rows_around_an_accumulations_end(tb, d, dtype):
    # tiles whose rows see 32768 keys, one more or one less: some rows have keys in the second segment
    from trellis_cpp_b200 import ops
    n = 33500
    g = torch.Generator(device="cuda").manual_seed(d)
    q, k, v = (torch.randn((n, 1, d), device="cuda", generator=g).to(dtype) for _ in range(3))
    _sampled(ops, q, k, v, [0, n], [0, n], [(0, t) for t in (0, 127, 32640, 32767, 32768, 32769, 32895, 33023, 33499)], True)
    k[32770] = math.nan                              # seen by the rows from 32770 on; the values there are numbers
    out = ops.attention(q, k, v, causal=True)
    assert bool(torch.isfinite(out[:32770]).all()) and bool(torch.isnan(out[32770:]).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [64, 128])
def test_sums_over_millions_of_keys(tb, d, dtype):
    """Equal weights (p = 1, exact) and values in [1, 2). An accumulation of 32768 keys is 2048 additions of
    16 products to the sum so far, each of the 17 cut by less than a step (2 half steps) of a sum that ends
    at its largest: at most 2048 * 34 half steps of it. The 128 segments add up in 128 more roundings."""
    from trellis_cpp_b200 import ops
    nk = 1 << 22
    nq = torch.cuda.get_device_properties(0).multi_processor_count * 128 * (d // 64)      # one range of keys
    g = torch.Generator(device="cuda").manual_seed(d)
    q = torch.zeros((nq, 1, d), dtype=dtype, device="cuda")
    k = torch.randn((nk, 1, d), device="cuda", generator=g).to(dtype)
    v = (1 + torch.rand((nk, 1, d), device="cuda", generator=g)).to(dtype)
    want = v.double().mean(0)
    out, lse = ops.attention(q, k, v, out_dtype=torch.float32, return_lse=True)
    ops.check_device()
    f = ref.HALF[torch.float32]
    assert float(((out[[0, 1, nq // 2, nq - 1]].double() - want).abs() / want).max()) <= (2048 * 34 + 2 * 128) * f
    assert bool((out == out[:1]).all())
    assert float((lse.double() - math.log(nk)).abs().max()) <= 2 ** -13 + (64 + 128) * f + 4 * f * math.log(nk)


def test_a_tile_of_seconds(tb):
    """450 million keys, 8 columns, on one tile an SM: each tile takes longer than the 4e9 cycles (2 s) that
    a wait may last, and no wait is as long as a tile."""
    from trellis_cpp_b200 import ops
    nk, nq = 450_000_000, torch.cuda.get_device_properties(0).multi_processor_count * 128
    q = torch.zeros((nq, 1, 8), dtype=torch.bfloat16, device="cuda")
    k = torch.zeros((nk, 1, 8), dtype=torch.bfloat16, device="cuda")
    v = torch.ones((nk, 1, 8), dtype=torch.bfloat16, device="cuda")
    v[nk // 2:] = 2.0
    a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    a.record()
    out = ops.attention(q, k, v, out_dtype=torch.float32)
    b.record()
    ops.check_device()
    f = ref.HALF[torch.float32]
    # segments of one value are exact (32768 and 65536); their 13733 sums round once each
    assert float((out - 1.5).abs().max()) <= 1.5 * 2 * 13734 * f
    print("ms:", a.elapsed_time(b))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("h,lg", [(150, 22), (1, 24)])
def test_new_token_sums_over_millions_of_keys(tb, h, lg, dtype):
    # as above; a warp's accumulation holds 32768 keys, and there are at most 32 in a row, 8 warps, 32 ranges
    from trellis_cpp_b200 import ops
    nk, d = (1 << lg) + 77, 8
    g = torch.Generator(device="cuda").manual_seed(lg)
    q = torch.zeros((1, h, d), dtype=dtype, device="cuda")
    k = torch.zeros((nk, h, d), dtype=dtype, device="cuda")
    v = (1 + torch.rand((nk, 1, d), device="cuda", generator=g)).to(dtype).expand(nk, h, d).contiguous()
    want = v[:, 0].double().mean(0)
    out, lse = ops.attention(q, k, v, out_dtype=torch.float32, return_lse=True)
    ops.check_device()
    f = ref.HALF[torch.float32]
    assert float(((out[0].double() - want).abs() / want).max()) <= (2048 * 34 + 2 * 300) * f
    assert float((lse.double() - math.log(nk)).abs().max()) <= 2 ** -13 + (64 + 512) * f + 4 * f * math.log(nk)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("order", ["flat", "rising", "falling"])
@pytest.mark.parametrize("h,d,nk", [(150, 8, 300003), (160, 72, 140001)])
def test_new_tokens_against_more_keys_than_one_accumulation_takes(tb, h, d, nk, order, dtype):
    from trellis_cpp_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(d)
    q = torch.randn((3, h, d), device="cuda", generator=g).to(dtype)
    k = torch.randn((nk, h, d), device="cuda", generator=g, dtype=dtype)
    v = torch.randn((nk, h, d), device="cuda", generator=g, dtype=dtype)
    if order != "flat":
        q, ramp = q.abs(), torch.linspace(0.1, 3, nk, device="cuda").to(dtype)[:, None, None]
        k.abs_().mul_(ramp if order == "rising" else ramp.flip(0))
    out = ops.attention(q, k, v, causal=True)
    ops.check_device()
    for a in (0, h - 1):
        want, _, wgt, reach = ref.attention(q[:, a:a + 1], k[:, a:a + 1], v[:, a:a + 1], [0, 3], [0, nk], True, d ** -0.5)
        assert ref.close(out[:, a:a + 1], want, ref.attention_tolerance(want, wgt, reach, d, nk, dtype, dtype)) <= 1.0
