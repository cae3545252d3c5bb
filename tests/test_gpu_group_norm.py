"""GroupNorm over packed sets (tb_group_norm) vs the 64-bit form. Tolerance per element, with z the
normalised value, f = 2^-24 and |mean| / std = r: the mean is rounded once (a share r of the step), the
difference, the factor (rstd, w and their product) and the sum with b take one rounding each, the
variance's share is below 64 f (batches of 4 rows joined up to a few hundred times in 32 bits, halved
by the root): (|z w| (70) + r |w| 2 + |b|) f. SiLU: its slope is at most 1.1, its exponential and
division add 8 f of the result (2 + 1.17 |y| steps of the fast exponential: up to |y| = 5 below 8) and
the result is rounded to the type."""
import math

import pytest
import torch

import packed_ref as ref

pytestmark = pytest.mark.gpu


def _inputs(seed, n, c, dtype, mean=0.5, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = (torch.randn((n, c), device="cuda", generator=g) * std + mean).to(dtype)
    w = 1 + 0.1 * torch.randn(c, device="cuda", generator=g)
    b = 0.1 * torch.randn(c, device="cuda", generator=g)
    return x, w, b


def _tolerance(x, groups, w, b, off, eps, act, out_dtype):
    f = ref.HALF[torch.float32]
    z = ref.group_norm(x, groups, None, None, off, eps, "none")
    aw = 1.0 if w is None else w.double().abs()
    ab = 0.0 if b is None else b.double().abs()
    r = torch.zeros_like(z)
    for s, e in zip(off, off[1:]):
        if e > s:
            y = x[s:e].double().view(e - s, groups, -1)
            m = y.mean((0, 2), keepdim=True)
            sd = torch.sqrt(((y - m) ** 2).mean((0, 2), keepdim=True) + eps)
            r[s:e] = (m.abs() / sd).expand_as(y).reshape(e - s, -1)
    t = (z.abs() * aw * 70 + 2 * r * aw + ab) * f
    if act == "silu":
        t = 1.1 * t + 16 * f * (z.abs() * aw + ab)
    y = ref.group_norm(x, groups, w, b, off, eps, act)
    return y, t + ref.HALF[out_dtype] * y.abs() + (2.0 ** -25 if out_dtype == torch.float16 else 1e-38)


def _check(ops, x, groups, w, b, off, eps=1e-5, act="none", out_dtype=None, out=None):
    got = ops.group_norm(x, groups, w, b, ref.table(off), eps=eps, act=act, out_dtype=out_dtype, out=out)
    ops.check_device()
    want, tol = _tolerance(x, groups, w, b, off, eps, act, got.dtype)
    assert ref.close(got, want, tol) <= 1.0
    return got


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("act", ["none", "silu"])
@pytest.mark.parametrize("lengths", [[1], [7], [800], [0, 3, 0, 0, 129, 1], [5000, 2, 333, 16, 17], [40000]])
def test_lengths(tb, lengths, act, dtype):
    from trellis_cpp_b200 import ops
    x, w, b = _inputs(len(lengths), sum(lengths), 64, dtype)
    _check(ops, x, 16, w, b, ref.offsets(lengths), act=act)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("c,groups", [(8, 1), (8, 8), (8, 2), (24, 3), (40, 5), (40, 4), (128, 32), (512, 32), (1000, 50),
                                      (2048, 32), (2048, 1), (2048, 2048), (264, 11)])
def test_channels_and_groups(tb, c, groups, dtype):
    from trellis_cpp_b200 import ops
    x, w, b = _inputs(c, 700, c, dtype)
    _check(ops, x, groups, w, b, [0, 100, 700])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_float32_output_and_no_affine(tb, dtype):
    from trellis_cpp_b200 import ops
    x, w, b = _inputs(2, 900, 96, dtype)
    a = _check(ops, x, 8, None, None, [0, 900], out_dtype=torch.float32)
    assert torch.equal(a.to(dtype), ops.group_norm(x, 8))
    _check(ops, x, 8, w, None, [0, 400, 900], act="silu", out_dtype=torch.float32)
    _check(ops, x, 8, None, b, [0, 400, 900])


@pytest.mark.parametrize("mean,std", [(100.0, 1.0), (1000.0, 0.1), (0.0, 1e-4), (0.0, 1e4)])
def test_means_far_from_zero(tb, mean, std):
    from trellis_cpp_b200 import ops
    x, w, b = _inputs(3, 6000, 32, torch.float32, mean, std)
    _check(ops, x, 4, w, b, [0, 6000])


def test_constant_and_outlier_sets(tb):
    from trellis_cpp_b200 import ops
    x = torch.full((300, 16), 3.0, device="cuda")
    got = ops.group_norm(x, 4)
    assert bool((got == 0).all())                    # variance 0: (x - mean) is 0
    x, w, b = _inputs(4, 3000, 16, torch.float32)
    x[0] = 1e4                                       # the first row is far off
    _check(ops, x, 4, w, b, [0, 3000])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_outside_the_sets(tb, dtype):
    from trellis_cpp_b200 import ops
    off = [11, 40, 40, 300]
    x, w, b = _inputs(5, 400, 64, dtype)
    x[:11], x[300:] = math.nan, math.inf
    out = torch.full((400, 64), 5.0, dtype=dtype, device="cuda")
    _check(ops, x, 8, w, b, off, act="silu", out=out)
    assert bool((out[:11] == 5).all()) and bool((out[300:] == 5).all())
    x[50, 3] = math.nan                              # one value: its set's group, nothing else
    got = ops.group_norm(x, 8, w, b, ref.table(off))
    assert bool(torch.isnan(got[40:300, :8]).all())
    assert bool(torch.isfinite(got[40:300, 8:]).all()) and bool(torch.isfinite(got[11:40]).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_in_place_and_repeats_to_the_bit(tb, dtype):
    from trellis_cpp_b200 import ops
    x, w, b = _inputs(6, 30000, 128, dtype)
    off = ref.table([0, 11000, 11001, 30000])
    want = ops.group_norm(x, 32, w, b, off, act="silu")
    for _ in range(3):
        assert torch.equal(want, ops.group_norm(x, 32, w, b, off, act="silu"))
    y = x.clone()
    assert ops.group_norm(y, 32, w, b, off, act="silu", out=y).data_ptr() == y.data_ptr() and torch.equal(y, want)


def test_many_sets(tb):
    from trellis_cpp_b200 import ops
    g = torch.Generator().manual_seed(1)
    lengths = torch.randint(0, 12, (3000,), generator=g).tolist()
    x, w, b = _inputs(7, sum(lengths), 32, torch.bfloat16)
    _check(ops, x, 4, w, b, ref.offsets(lengths), eps=1e-3)


def test_captured_call_follows_its_table(tb):
    from trellis_cpp_b200 import ops
    x, w, b = _inputs(8, 5000, 64, torch.bfloat16)
    off = ref.table([0, 100, 5000])
    ops.group_norm(x, 8, w, b, off)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for act in ("none", "silu"):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(ops.group_norm(x, 8, w, b, off, act=act))
        graphs.append(gr)
    off.copy_(ref.table([0, 3001, 5000]))
    torch.cuda.synchronize()
    for _ in range(3):
        for gr in graphs:
            with torch.cuda.stream(torch.cuda.Stream()):
                gr.replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], ops.group_norm(x, 8, w, b, off))
    assert torch.equal(outs[1], ops.group_norm(x, 8, w, b, off, act="silu"))


def test_more_than_2_31_elements(tb):
    from trellis_cpp_b200 import ops
    n, c = 1100000, 2048                             # 2.25e9 elements, 4.5 GB each way
    x = torch.zeros((n, c), dtype=torch.bfloat16, device="cuda")
    part, w, b = _inputs(9, 1000, c, torch.bfloat16)
    x[-1000:] = part
    y = ops.group_norm(x, 32, w, None, ref.table([0, n - 1000, n]))
    want, tol = _tolerance(part, 32, w, None, [0, 1000], 1e-5, "none", torch.bfloat16)
    assert ref.close(y[-1000:], want, tol) <= 1.0
    assert int(y[:-1000].count_nonzero()) == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_thousands_of_small_sets_in_three_passes(tb, dtype):
    from trellis_cpp_b200 import ops
    g = torch.Generator().manual_seed(3)
    lengths = torch.randint(0, 9, (2000,), generator=g).tolist()
    lengths[700], lengths[1999] = 1300, 0
    off = ref.offsets(lengths, 100)
    x, w, b = _inputs(12, off[-1] + 50, 64, dtype)
    x[:100] = float("nan")
    x[off[-1]:] = float("nan")
    y = torch.full_like(x, 3.0)
    _check(ops, x, 8, w, b, off, eps=1e-3, act="silu", out=y)
    assert bool((y[:100] == 3).all()) and bool((y[off[-1]:] == 3).all())


@pytest.mark.parametrize("off", [[0, 6000, 3000, 10000], [-3, 5000, 10000, 10000], [0, 50, 100, 17000]])
def test_bad_tables_of_long_arrays_are_reported(tb, off):
    from trellis_cpp_b200 import ops
    x, w, b = _inputs(13, 10000, 32, torch.bfloat16)
    ops.group_norm(x, 4, w, b, ref.table(off))
    with pytest.raises(ops.TBError) as e:
        ops.check_device()
    assert e.value.status == 5 and "offset table" in str(e.value)
    _check(ops, x, 4, w, b, [0, 5000, 10000])


@pytest.mark.parametrize("off", [[0, 60, 30, 100], [-3, 50, 100, 100], [0, 50, 100, 170]])
def test_bad_tables_are_reported(tb, off):
    from trellis_cpp_b200 import ops
    x, w, b = _inputs(10, 100, 32, torch.float32)
    ops.group_norm(x, 4, w, b, ref.table(off))
    with pytest.raises(ops.TBError) as e:
        ops.check_device()
    assert e.value.status == 5 and "offset table" in str(e.value)
    _check(ops, x, 4, w, b, [0, 50, 100])


def test_refusals(tb):
    from trellis_cpp_b200 import ops
    x, w, b = _inputs(11, 10, 32, torch.bfloat16)
    for call, kind in [
        (lambda: ops.group_norm(x.cpu(), 4), ValueError),
        (lambda: ops.group_norm(x[:, ::2], 4), ValueError),
        (lambda: ops.group_norm(x, 4, w[:16]), ValueError),
        (lambda: ops.group_norm(x, 4, w.double()), ValueError),
        (lambda: ops.group_norm(x, 4, offsets=ref.table([0, 10]).long()), ValueError),
        (lambda: ops.group_norm(x, 4, out=torch.empty_like(x)[:5]), ValueError),
        (lambda: ops.group_norm(x, 5), ops.TBError),
        (lambda: ops.group_norm(x, 0), ops.TBError),
        (lambda: ops.group_norm(x, 4, eps=-1.0), ops.TBError),
        (lambda: ops.group_norm(x, 4, out_dtype=torch.float16), ops.TBError),
        (lambda: ops.group_norm(torch.zeros((4, 20), device="cuda"), 4), ops.TBError),
    ]:
        with pytest.raises(kind):
            call()
    assert ops.group_norm(x[:0], 4).shape == (0, 32)
    assert ops.group_norm(x, 4, offsets=ref.table([0])).shape == x.shape
