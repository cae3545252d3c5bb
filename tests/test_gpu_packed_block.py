"""The packed-set operators as a transformer block uses them: LayerNorm, q|k|v product, rotary
positions from the voxels' coordinates, attention, output product with the residual, and GroupNorm
with SiLU of the result, against the same block in 64 bits."""
import pytest
import torch

import packed_ref as ref

pytestmark = pytest.mark.gpu


def _block(ops, x, coords, off, wn, bn, wqkv, wo, gw, gb, h, hk, d):
    n = x.shape[0]
    y = ops.layer_norm(x, wn, bn)
    qkv = ops.linear(y, wqkv).view(n, h + 2 * hk, d)
    ops.rope(qkv[:, :h + hk], coords, (d // 6,) * 3, out=qkv[:, :h + hk])
    a = ops.attention(qkv[:, :h], qkv[:, h:h + hk], qkv[:, h + hk:], off)
    z = ops.linear(a.view(n, h * d), wo, residual=x)
    return ops.group_norm(z, 16, gw, gb, off, act="silu")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("h,hk,d", [(4, 4, 64), (4, 2, 128)])
def test_block(tb, h, hk, d, dtype):
    from trellis_cpp_b200 import ops
    lengths = [600, 1, 333]
    off, n, c = ref.offsets(lengths), sum(lengths), 256
    g = torch.Generator(device="cuda").manual_seed(h + d)

    def rnd(*s, scale=1.0, mean=0.0, dt=dtype):
        return (torch.randn(s, device="cuda", generator=g) * scale + mean).to(dt)

    x = rnd(n, c)
    coords = torch.randint(0, 64, (n, 4), device="cuda", generator=g, dtype=torch.int32)
    wn, bn = rnd(c, scale=0.1, mean=1.0, dt=torch.float32), rnd(c, scale=0.1, dt=torch.float32)
    wqkv, wo = rnd((h + 2 * hk) * d, c, scale=c ** -0.5), rnd(c, h * d, scale=(h * d) ** -0.5)
    gw, gb = rnd(c, scale=0.1, mean=1.0, dt=torch.float32), rnd(c, scale=0.1, dt=torch.float32)
    args = (x, coords, ref.table(off), wn, bn, wqkv, wo, gw, gb, h, hk, d)
    out = _block(ops, *args)
    ops.check_device()

    xd = x.double()
    y = (xd - xd.mean(1, keepdim=True)) / torch.sqrt(xd.var(1, correction=0, keepdim=True) + 1e-6) * wn.double() + bn.double()
    qkv = (y @ wqkv.double().T).view(n, h + 2 * hk, d)
    qk = ref.rope(qkv[:, :h + hk], coords[:, 1:], (d // 6,) * 3, 10000.0, "pairs", False, False)
    a, _, _, _ = ref.attention(qk[:, :h], qk[:, h:], qkv[:, h + hk:], off, off, False, d ** -0.5)
    want = ref.group_norm(a.reshape(n, h * d) @ wo.double().T + xd, 16, gw, gb, off, 1e-5, "silu")
    # seven roundings to the type on the way (y, qkv, rope, p, a, z, out), each a relative half step of
    # values of the result's size; 8 of them allow for sums that partly cancel
    half = ref.HALF[dtype] if dtype != torch.float32 else 2.0 ** -19
    err = (out.double() - want).norm() / want.norm()
    assert float(err) <= 8 * half

    # captured and replayed on other inputs
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        held = _block(ops, *args)
    x.copy_(rnd(n, c))
    gr.replay()
    torch.cuda.synchronize()
    assert torch.equal(held, _block(ops, *args))
