"""Pairs behind the last section (tb_rope) keep their bits: infinities, values that are no number with
their payload, and zeros of either sign, whole 16-byte words of them or the rest of a word that also
holds pairs that turn."""
import pytest
import torch

import packed_ref as ref

pytestmark = pytest.mark.gpu

# as the type's bits: inf, -inf, a quiet and a signalling NaN with payloads, -NaN, -0, +0, the smallest step
BITS = {torch.bfloat16: [0x7F80, 0xFF80, 0x7FC5, 0x7F83, 0xFFC1, 0x8000, 0x0000, 0x0001],
        torch.float16: [0x7C00, 0xFC00, 0x7E35, 0x7C03, 0xFE01, 0x8000, 0x0000, 0x0001],
        torch.float32: [0x7F800000, 0xFF800000, 0x7FC00305, 0x7F800003, 0xFFC00001, 0x80000000, 0, 1]}


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("layout", ["pairs", "halves"])
@pytest.mark.parametrize("d,sections", [(8, (1,)), (16, (2, 1)), (24, (5,)), (64, (10, 10, 7)), (64, (1,)), (128, (21, 21, 21)),
                                        (128, (9, 8)), (256, (50, 51))])
def test_kept_pairs_keep_their_bits(tb, d, sections, layout, dtype):
    from trellis_cpp_b200 import ops
    n, h, half, turned = 37, 5, d // 2, sum(sections)
    word = torch.int16 if dtype != torch.float32 else torch.int32
    span = 1 << (8 * word.itemsize)
    vals = torch.tensor([b - span if b >= span // 2 else b for b in BITS[dtype]], dtype=word, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(d + turned)
    x = torch.randn((n, h, d), device="cuda", generator=g).to(dtype)
    kept = torch.zeros(d, dtype=torch.bool, device="cuda")
    if layout == "pairs":
        kept[2 * turned:] = True
    else:
        kept[turned:half] = kept[half + turned:] = True
    odd = vals[torch.randint(0, len(vals), (n, h, d), device="cuda", generator=g)]
    bits = torch.where(kept, odd, x.view(word))
    x = bits.view(dtype)
    pos = torch.randint(-50, 1000, (n, len(sections)), device="cuda", generator=g, dtype=torch.int32)
    plain = torch.where(kept, torch.zeros_like(x), x)
    for inverse in (False, True):
        got = ops.rope(x, pos, sections, layout=layout, inverse=inverse)
        assert torch.equal(got.view(word)[..., kept], bits[..., kept])
        # the pairs that turn: the same to the bit as beside zeros
        want = ops.rope(plain, pos, sections, layout=layout, inverse=inverse)
        assert torch.equal(got[..., ~kept], want[..., ~kept])
        exact = ref.rope(plain, pos, sections, 10000.0, layout, False, inverse)
        half_steps = ref.HALF[dtype] * exact.abs() + 11 * ref.HALF[torch.float32] * 8 + 2.0 ** -25   # pairs are shorter than 8
        assert ref.close(want, exact, half_steps) <= 1.0
    again = x.clone()
    ops.rope(again, pos, sections, layout=layout, out=again)
    assert torch.equal(again.view(word)[..., kept], bits[..., kept])
