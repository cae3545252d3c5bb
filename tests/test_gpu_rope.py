"""Rotary positions (tb_rope) vs the 64-bit form. Tolerance per element: the two products and their
sum in 32 bits (3 half steps), sine and cosine of a reduced angle in 32 bits (the angle's rounding
pi * 2^-24 and 2 half steps of the function each: 8 half steps together), all relative to the pair's
length sqrt(a^2 + b^2), and the rounding to the output's type."""
import pytest
import torch

import packed_ref as ref

pytestmark = pytest.mark.gpu


def _check(ops, x, coords, sections, layout="pairs", joint=False, inverse=False, theta=10000.0, out=None):
    pos = coords[:, -len(sections):]
    want = ref.rope(x, pos, sections, theta, layout, joint, inverse)
    got = ops.rope(x, coords, sections, theta=theta, layout=layout, freqs="joint" if joint else "axis", inverse=inverse, out=out)
    half = x.shape[2] // 2
    y = x.double()
    if layout == "pairs":
        length = torch.hypot(y[..., 0::2], y[..., 1::2]).repeat_interleave(2, -1)
    else:
        length = torch.hypot(y[..., :half], y[..., half:]).repeat(1, 1, 2)
    tol = ref.HALF[x.dtype] * want.abs() + 11 * ref.HALF[torch.float32] * length + 1e-38
    if x.dtype == torch.float16:
        tol = tol + 2.0 ** -25                       # half the smallest step of float16
    assert ref.close(got, want, tol) <= 1.0
    kept = 2 * sum(sections) if layout == "pairs" else None
    if layout == "pairs":
        assert torch.equal(got[..., kept:], x[..., kept:])
    else:
        s = sum(sections)
        assert torch.equal(got[..., s:half], x[..., s:half]) and torch.equal(got[..., half + s:], x[..., half + s:])
    return got


def _x(seed, n, h, d, dtype):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn((n, h, d), device="cuda", generator=g).to(dtype)


def _pos(seed, n, axes, lo, hi):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(lo, hi, (n, axes), device="cuda", generator=g, dtype=torch.int32)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("layout", ["pairs", "halves"])
@pytest.mark.parametrize("d,sections", [(8, (4,)), (8, (1, 1, 1)), (24, (3, 4, 5)), (40, (6, 6, 6)), (64, (10, 10, 10)),
                                        (128, (21, 21, 21)), (128, (16, 24, 24)), (128, (16, 16, 16, 16)), (256, (128,))])
def test_head_dims_and_sections(tb, d, sections, layout, dtype):
    from trellis_cpp_b200 import ops
    x = _x(d, 77, 3, d, dtype)
    for joint in (False, True):
        for inverse in (False, True):
            _check(ops, x, _pos(d, 77, len(sections), 0, 1024), sections, layout, joint, inverse)


@pytest.mark.parametrize("n,h", [(1, 1), (1, 7), (5, 64), (257, 5), (4000, 24)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_and_heads(tb, n, h, dtype):
    from trellis_cpp_b200 import ops
    _check(ops, _x(n, n, h, 64, dtype), _pos(n, n, 3, 0, 512), (10, 10, 10))


@pytest.mark.parametrize("lo,hi", [(-1000, 0), (100000, 1 << 20), (-(1 << 31), (1 << 31) - 1)])
def test_far_and_negative_positions(tb, lo, hi):
    from trellis_cpp_b200 import ops
    n = 500
    x, pos = _x(1, n, 2, 128, torch.float32), _pos(2, n, 3, lo, hi)
    # in 64 bits the angle itself is off by half a step of up to 2^31: 2^31 * 2^-53, and as much for the
    # frequency and for the reference's: 4 * 2^-22 at the farthest
    want = ref.rope(x, pos, (21, 21, 21), 10000.0, "pairs", False, False)
    got = ops.rope(x, pos, (21, 21, 21))
    y = x.double()
    length = torch.hypot(y[..., 0::2], y[..., 1::2]).repeat_interleave(2, -1)
    far = max(abs(lo), abs(hi))
    tol = ref.HALF[torch.float32] * want.abs() + (11 * ref.HALF[torch.float32] + 4 * far * 2.0 ** -53) * length
    assert ref.close(got, want, tol) <= 1.0


@pytest.mark.parametrize("layout", ["pairs", "halves"])
def test_voxel_rows_with_batch_in_views_and_in_place(tb, layout):
    from trellis_cpp_b200 import ops
    n, h, d = 301, 4, 64
    qkv = _x(3, n, 3 * h, d, torch.bfloat16)
    keep = qkv.clone()
    coords = _pos(4, n, 4, 0, 64)                    # (b, x, y, z): the batch has no part in it
    want = _check(ops, qkv[:, :2 * h], coords, (10, 10, 10), layout)
    ops.rope(qkv[:, :2 * h], coords, (10, 10, 10), layout=layout, out=qkv[:, :2 * h])
    assert torch.equal(qkv[:, :2 * h], want) and torch.equal(qkv[:, 2 * h:], keep[:, 2 * h:])
    hm = keep.transpose(0, 1).contiguous().transpose(0, 1)         # [heads][rows][dim] memory
    assert torch.equal(ops.rope(hm[:, :2 * h], coords, (10, 10, 10), layout=layout), want)


@pytest.mark.parametrize("layout", ["pairs", "halves"])
@pytest.mark.parametrize("joint", [False, True])
def test_inverse_is_the_gradient(tb, layout, joint):
    """y = R x is linear: <R dx, u> = <dx, R^T u> for the inverse's u, and differences of <y, u> along
    each coordinate of a row agree with it (exactly linear, so any step will do)."""
    from trellis_cpp_b200 import ops
    fr = "joint" if joint else "axis"
    x, pos = _x(5, 9, 2, 24, torch.float32), _pos(6, 9, 2, 0, 300)
    u = _x(7, 9, 2, 24, torch.float32)
    grad = ops.rope(u, pos, (5, 6), layout=layout, freqs=fr, inverse=True).double()
    base = (ops.rope(x, pos, (5, 6), layout=layout, freqs=fr).double() * u.double()).sum((1, 2))
    for d in range(24):
        dx = torch.zeros_like(x)
        dx[:, 1, d] = 1.0
        diff = (ops.rope(x + dx, pos, (5, 6), layout=layout, freqs=fr).double() * u.double()).sum((1, 2)) - base
        # x + dx, and each of 48 products, rounded relative to values below 6: 60 half steps of 36
        assert float((diff - grad[:, 1, d]).abs().max()) <= 60 * 36 * ref.HALF[torch.float32]
    back = ops.rope(ops.rope(x, pos, (5, 6), layout=layout, freqs=fr), pos, (5, 6), layout=layout, freqs=fr, inverse=True)
    assert float((back - x).abs().max()) <= 2 * 12 * ref.HALF[torch.float32] * 6


def test_captured(tb):
    from trellis_cpp_b200 import ops
    x, pos = _x(8, 100, 4, 64, torch.bfloat16), _pos(9, 100, 3, 0, 64)
    ops.rope(x, pos, (10, 10, 10))
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        y = ops.rope(x, pos, (10, 10, 10))
    x.copy_(_x(10, 100, 4, 64, torch.bfloat16))
    pos.copy_(_pos(11, 100, 3, 0, 64))
    gr.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, ops.rope(x, pos, (10, 10, 10)))


def test_more_than_2_31_elements(tb):
    from trellis_cpp_b200 import ops
    n, h, d = 140000, 128, 128                       # 2.3e9 elements, 4.6 GB each way
    x = torch.zeros((n, h, d), dtype=torch.bfloat16, device="cuda")
    pos = _pos(12, n, 3, 0, 1024)
    x[-50:] = _x(13, 50, h, d, torch.bfloat16)
    y = ops.rope(x, pos, (21, 21, 21))
    assert torch.equal(y[-50:], ops.rope(x[-50:].contiguous(), pos[-50:].contiguous(), (21, 21, 21)))
    assert int(y[:-50].count_nonzero()) == 0


def test_refusals(tb):
    from trellis_cpp_b200 import ops
    x, pos = _x(1, 10, 2, 64, torch.bfloat16), _pos(1, 10, 3, 0, 9)
    for call, kind in [
        (lambda: ops.rope(x.cpu(), pos, (10, 10, 10)), ValueError),
        (lambda: ops.rope(x, pos.long(), (10, 10, 10)), ValueError),
        (lambda: ops.rope(x, pos[:5], (10, 10, 10)), ValueError),
        (lambda: ops.rope(x, pos, (10,)), ValueError),
        (lambda: ops.rope(x, pos, ()), ValueError),
        (lambda: ops.rope(x, pos, (10, 10, 10), layout="thirds"), ValueError),
        (lambda: ops.rope(x, pos, (10, 10, 10), freqs="none"), ValueError),
        (lambda: ops.rope(x, pos, (10, 10, 10), out=torch.empty_like(x).float()), ValueError),
        (lambda: ops.rope(x, pos, (11, 11, 11)), ops.TBError),            # 33 pairs in a head of 32
        (lambda: ops.rope(x, pos, (0, 10, 10)), ops.TBError),
        (lambda: ops.rope(x, pos, (10, 10, 10), theta=0.0), ops.TBError),
        (lambda: ops.rope(x[..., :60], pos, (10, 10, 10)), ops.TBError),  # head_dim % 8
        (lambda: ops.rope(x, pos, (10, 10, 10), out=x[:1].expand(10, 2, 64)), ops.TBError),
    ]:
        with pytest.raises(kind):
            call()
    assert ops.rope(x[:0], pos[:0], (10, 10, 10)).shape == (0, 2, 64)
