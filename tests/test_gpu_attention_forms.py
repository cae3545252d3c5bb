"""Forms of attention (tb_attention) beside those of test_gpu_attention.py: sets that CTA pairs take with
heads of 72 to 120 columns, whose second half of V is partly behind the head's end; caches that grow in
place; hundreds of sets in 128-row tiles; rows that see one key."""
import math

import pytest
import torch

import packed_ref as ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("out_dtype", [None, torch.float32])
@pytest.mark.parametrize("d", [72, 80, 88, 96, 104, 112, 120])
@pytest.mark.parametrize("h,hk,ql,kl", [(2, 2, [300, 0, 257], [333, 40, 129]), (6, 2, [129, 400], [700, 100])])
def test_pairs_of_partly_filled_heads(tb, h, hk, ql, kl, d, causal, out_dtype, dtype):
    """Rows an average set of more than a tile's tokens (128 / heads a key head): pairs."""
    from trellis_cpp_b200 import ops
    assert -(-sum(ql) // len(ql)) > 128 // (h // hk)
    g = torch.Generator(device="cuda").manual_seed(d)
    wide = torch.randn((sum(kl), hk, 136), device="cuda", generator=g).to(dtype)
    wide[..., d:] = math.nan                         # behind a head's last column: not read
    q = torch.randn((sum(ql), h, d), device="cuda", generator=g).to(dtype)
    k, v = wide[..., :d], torch.randn((sum(kl), hk, d), device="cuda", generator=g).to(dtype)
    qo, ko = ref.offsets(ql), ref.offsets(kl)
    got = torch.full((sum(ql), h, 136), 9.0, dtype=out_dtype or dtype, device="cuda")
    out, lse = ops.attention(q, k, v, ref.table(qo), ref.table(ko), causal=causal, out=got[..., :d], return_lse=True)
    ops.check_device()
    want, wlse, wgt, reach = ref.attention(q, k, v, qo, ko, causal, d ** -0.5)
    tol = ref.attention_tolerance(want, wgt, reach, d, max(kl), dtype, out.dtype)
    assert ref.close(out, want, tol) <= 1.0 and bool((got[..., d:] == 9).all())
    none = wlse == -math.inf
    assert bool((lse[none] == -math.inf).all()) and bool((out[none] == 0).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_caches_that_grow_in_place(tb, dtype):
    """Each sequence has room for 600 keys in one buffer. The tables name two sets a sequence, its keys and
    its spare rows, the latter without queries; a step writes the new key and raises one entry."""
    from trellis_cpp_b200 import ops
    room, lengths, h, hk, d = 600, [17, 599, 1, 300], 8, 2, 64
    b = len(lengths)
    g = torch.Generator(device="cuda").manual_seed(1)
    k = torch.full((b * room, hk, d), math.nan, dtype=dtype, device="cuda")      # spare rows hold no numbers
    v = torch.full((b * room, hk, d), math.inf, dtype=dtype, device="cuda")
    for s, n in enumerate(lengths):
        k[s * room:s * room + n] = torch.randn((n, hk, d), device="cuda", generator=g).to(dtype)
        v[s * room:s * room + n] = torch.randn((n, hk, d), device="cuda", generator=g).to(dtype)
    q_off = ref.table([x for s in range(b) for x in (s, s + 1)] + [b])           # 0 1 | 1 1 | 1 2 | ...
    k_off = ref.table([x for s, n in enumerate(lengths) for x in (s * room, s * room + n)] + [b * room])
    for _ in range(2):
        q = torch.randn((b, h, d), device="cuda", generator=g).to(dtype)
        out = ops.attention(q, k, v, q_off, k_off)
        ops.check_device()
        for s, n in enumerate(lengths):
            at = slice(s * room, s * room + n)
            want, _, wgt, reach = ref.attention(q[s:s + 1], k[at], v[at], [0, 1], [0, n], False, d ** -0.5)
            assert ref.close(out[s:s + 1], want, ref.attention_tolerance(want, wgt, reach, d, n, dtype, dtype)) <= 1.0
        rows = k_off[1::2].long()
        k[rows] = torch.randn((b, hk, d), device="cuda", generator=g).to(dtype)
        v[rows] = torch.randn((b, hk, d), device="cuda", generator=g).to(dtype)
        k_off[1::2] += 1
        lengths = [n + 1 for n in lengths]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,top,h,hk,d,start", [(33, 400, 2, 2, 64, 0), (300, 200, 4, 2, 128, 7), (1500, 90, 2, 2, 64, 300),
                                                (700, 300, 1, 1, 128, 0)])
def test_many_sets_of_many_rows(tb, n, top, h, hk, d, start, dtype):
    """More sets than the tiles' list holds at once (32), empty ones among them, in 128-row tiles and pairs:
    each CTA takes over tiles from all over the table."""
    from trellis_cpp_b200 import ops
    g = torch.Generator().manual_seed(n)
    ql = (torch.randint(0, top, (n,), generator=g) * (torch.rand(n, generator=g) < 0.8)).tolist()
    kl = (torch.randint(0, top, (n,), generator=g) * (torch.rand(n, generator=g) < 0.9)).tolist()
    assert sum(ql) / n * (h // hk) > 17
    gd = torch.Generator(device="cuda").manual_seed(n)
    qo, ko = ref.offsets(ql, start), ref.offsets(kl)
    q = torch.randn((qo[-1] + 50, h, d), device="cuda", generator=gd).to(dtype)
    k = torch.randn((ko[-1], hk, d), device="cuda", generator=gd).to(dtype)
    v = torch.randn((ko[-1], hk, d), device="cuda", generator=gd).to(dtype)
    for causal in (False, True):
        out = torch.full(q.shape, 4.0, dtype=dtype, device="cuda")
        ops.attention(q, k, v, ref.table(qo), ref.table(ko), causal=causal, out=out)
        ops.check_device()
        want, _, wgt, reach = ref.attention(q, k, v, qo, ko, causal, d ** -0.5)
        assert ref.close(out, want, ref.attention_tolerance(want, wgt, reach, d, max(kl), dtype, dtype)) <= 1.0
        assert bool((out[:start] == 4).all()) and bool((out[qo[-1]:] == 4).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,h,hk,d", [(40, 2, 2, 64), (300, 2, 2, 64), (300, 4, 2, 128), (40, 1, 1, 72), (1, 4, 2, 128), (3, 8, 2, 64)])
def test_one_key_gives_its_value(tb, rows, h, hk, d, dtype):
    """The softmax of one score is 1: the value itself, to the bit. p and its sum are off by 2^-20 at most
    (scores below 2^4), far less than the half step within which the quotient rounds to the value. So for
    sets of one key, and for the first row of a causal set."""
    from trellis_cpp_b200 import ops
    sets = 6
    g = torch.Generator(device="cuda").manual_seed(rows + d)
    q = torch.randn((sets * rows, h, d), device="cuda", generator=g).to(dtype)
    k = torch.randn((sets, hk, d), device="cuda", generator=g).to(dtype)
    v = torch.randn((sets, hk, d), device="cuda", generator=g).to(dtype)
    qo = ref.table(list(range(0, sets * rows + 1, rows)))
    out = ops.attention(q, k, v, qo, ref.table(list(range(sets + 1))))
    want = v.repeat_interleave(h // hk, 1).repeat_interleave(rows, 0)
    assert torch.equal(out, want)
    k = torch.randn((sets * rows, hk, d), device="cuda", generator=g).to(dtype)
    v = torch.randn((sets * rows, hk, d), device="cuda", generator=g).to(dtype)
    out = ops.attention(q, k, v, qo, causal=True)
    assert torch.equal(out[::rows], v[::rows].repeat_interleave(h // hk, 1))
    ops.check_device()
