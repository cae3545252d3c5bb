"""Attention (tb_attention) at the ends of what scores and lengths may be: rows whose scores are all
-inf, in calls whose keys are cut into ranges and in others. The tolerance is that of
packed_ref.attention_tolerance."""
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
