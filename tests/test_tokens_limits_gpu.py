"""GPU: the token operators at the edges of what they take -- torch's default type, layouts with long strides, values near the type's largest."""
import math

import pytest
import torch

from tests import token_ref as R
from tests.conftest import rel_err

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF16 = torch.float32, torch.bfloat16


def rn(seed, *shape, dtype=F32, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g, dtype=F32) * scale).to(dtype)


@pytest.mark.parametrize("default", [BF16, torch.float64])
def test_results_do_not_depend_on_the_default_type(default):
    """The same bits under any torch default type: statistics and parameter gradients are fp32 buffers whatever it is."""
    from pdae_amd import tokens
    x, dy, w, b = (t.to(DEV) for t in (rn(1, 37, 72, dtype=BF16), rn(2, 37, 72, dtype=BF16), rn(3, 72), rn(4, 72)))
    q, k, v, g = (rn(5 + i, 2, 50, 2, 32, dtype=BF16).to(DEV) for i in range(4))

    def run():
        leaves = [t.clone().requires_grad_(True) for t in (x, w, b, q, k, v)]
        y = tokens.layer_norm(*leaves[:3])
        o = tokens.attention(*leaves[3:], causal=True)
        torch.autograd.backward([y, o], [dy, g])
        return [y.detach(), o.detach()] + [t.grad for t in leaves]
    want = run()
    before = torch.get_default_dtype()
    torch.set_default_dtype(default)
    try:
        got = run()
    finally:
        torch.set_default_dtype(before)
    for a, c in zip(want, got):
        assert a.dtype == c.dtype and torch.equal(a, c)


def test_single_token_queries_with_the_samples_inside_the_token():
    """[1, B, H, D] seen as [B, 1, H, D]: dense, with a token stride that no address uses."""
    from pdae_amd import tokens
    base = rn(1, 1, 512, 32, 128, dtype=BF16)
    k, v = rn(2, 512, 3, 8, 128, dtype=BF16), rn(3, 512, 3, 8, 128, dtype=BF16)
    q = base.to(DEV).transpose(0, 1)
    assert q.stride(1) == 1 << 21 and q.is_contiguous()
    kd, vd = k.to(DEV), v.to(DEV)
    plain = torch.empty(512, 1, 32, 128, dtype=BF16, device=DEV).copy_(q)
    assert plain.stride(1) == 4096
    got = tokens.attention(q, kd, vd)
    assert torch.equal(got, tokens.attention(plain, kd, vd))
    some = slice(200, 203)
    R.within(got[some], R.attention(base[0, some, None], k[some], v[some])["o"], "o")
    leaves = [t.clone().requires_grad_(True) for t in (q, kd, vd)]
    tokens.attention(*leaves).backward(torch.ones_like(got))
    want = [t.clone().requires_grad_(True) for t in (plain, kd, vd)]
    tokens.attention(*want).backward(torch.ones_like(got))
    assert all(torch.equal(a.grad, b.grad) for a, b in zip(leaves, want))


def test_head_major_caches_are_read_in_place():
    """[B, H, T, D] caches with T D = 2^20 (head strides far beyond the token limit): the bits of the token-major copy, and no copy of the cache."""
    from pdae_amd import tokens
    B, Hq, Hkv, T, D = 2, 16, 4, 8192, 128
    k, v, q = rn(1, B, Hkv, T, D, dtype=BF16), rn(2, B, Hkv, T, D, dtype=BF16), rn(3, B, Hq, 1, D, dtype=BF16)
    lens = torch.tensor([8192, 777], dtype=torch.int32, device=DEV)
    kd, vd, qd = (t.to(DEV).transpose(1, 2) for t in (k, v, q))
    want = tokens.attention(qd.contiguous(), kd.contiguous(), vd.contiguous(), k_len=lens, causal=True)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    got = tokens.attention(qd, kd, vd, k_len=lens, causal=True)
    assert torch.cuda.max_memory_allocated() - before < k.numel() * 2 // 4
    assert torch.equal(got, want)
    one = R.attention(q[1:].transpose(1, 2), k[1:, :, :777].transpose(1, 2), v[1:, :, :777].transpose(1, 2))["o"]
    R.within(got[1:], one, "o")
    leaves = [t.detach().requires_grad_(True) for t in (qd[:, :, :4], kd[:, :, :1], vd[:, :, :1])]      # gradients in the same layout
    tokens.attention(*leaves, k_len=lens).sum().backward()
    dense = [t.detach().contiguous().requires_grad_(True) for t in leaves]
    tokens.attention(*dense, k_len=lens).sum().backward()
    assert all(torch.equal(a.grad, b.grad) for a, b in zip(leaves, dense))


@pytest.mark.parametrize("B,Tq,Tk,Hq,Hkv,D,dtype", [(2, 40, 300, 2, 1, 32, F32), (1, 70, 300, 1, 1, 21, F32), (2, 200, 300, 2, 2, 128, BF16), (1, 150, 300, 1, 1, 13, BF16),
                                                    (4, 256, 300, 64, 64, 32, BF16), (2, 1, 300, 8, 2, 64, BF16), (1, 1, 6000, 4, 1, 128, BF16), (1, 3, 6000, 2, 1, 64, F32)])
def test_values_near_the_types_largest_while_the_scores_grow(B, Tq, Tk, Hq, Hkv, D, dtype):
    """Scores rise by 20 (29 powers of two) from the first key tile to the last and the values are 1e37 .. 3e38: the weights sum to one, so every output
    is finite, whatever reference the running sums are kept against."""
    from pdae_amd import tokens
    q, k = rn(1, B, Tq, Hq, D, scale=0.1), rn(2, B, Tk, Hkv, D, scale=0.1)
    q[..., 0], k[..., 0] = 4.0, (torch.arange(Tk) * (5.0 / Tk))[None, :, None]
    v = rn(3, B, Tk, Hkv, D).clamp(-3, 3) * 1e38
    g = rn(4, B, Tq, Hq, D, scale=1e-20)
    q, k, v, g = (t.to(dtype) for t in (q, k, v, g))
    assert torch.isfinite(v.float()).all()
    ref = R.attention(q, k, v, scale=1.0, d_o=g)
    leaves = [t.to(DEV).requires_grad_(True) for t in (q, k, v)]
    o = tokens.attention(*leaves, scale=1.0)
    o.backward(g.to(DEV))
    R.within(o, ref["o"], "o")
    for name, t in zip(("dq", "dk", "dv"), leaves):
        R.within(t.grad, ref[name], name)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,C", [(300, 64), (1100, 71), (33, 520), (1500, 1536), (5, 4099), (7, 16384), (5, 16391), (3, 40000)])
def test_layer_norm_in_place_is_the_same_bits(rows, C, dtype):
    from pdae_amd import hip as H
    k = H.DTYPES[dtype]
    x = rn(1, rows, C + 5, dtype=dtype).to(DEV)
    g, b = rn(2, C).to(DEV), rn(3, C).to(DEV)
    y, m, r = torch.empty_like(x), torch.empty(rows, device=DEV), torch.empty(rows, device=DEV)
    y.copy_(x)
    H.run(H.op_layernorm_fwd(x, g, b, rows, C, 1e-5, y, m, r, dtype=k, ldx=C + 5, ldy=C + 5))
    R.within(y[:, :C], R.layer_norm(x[:, :C].cpu(), g.cpu(), b.cpu(), 1e-5)["y"], "y")
    H.run(H.op_layernorm_fwd(x, g, b, rows, C, 1e-5, x, dtype=k, ldx=C + 5, ldy=C + 5))
    assert torch.equal(x, y)                                    # what lies between the rows included


@pytest.mark.parametrize("Tq,Tk,Hq,Hkv,D,causal", [(300, 700, 4, 2, 128, False), (700, 700, 4, 1, 72, True), (200, 1500, 2, 2, 32, True), (130, 600, 2, 1, 45, False), (64, 128, 2, 2, 64, False)])
def test_dq_of_bf16_tensors_is_little_more_than_its_own_rounding(Tq, Tk, Hq, Hkv, D, causal):
    """The norm of dq's error against the exact dq's, beside that of the exact dq rounded once to bf16 (e ~ 1.65e-3).  What comes on top: delta from the rounded o, at
    most the same relative size as the rounding of o against the largest part of dS: below e / 2 in these cases; dS in two planes leaves 2^-17.  In squares 1.25 e;
    with dS rounded to one plane (another e) it is above 1.41."""
    from pdae_amd import tokens
    q, k, v, g = (rn(i, 2, T, Hh, D, dtype=BF16) for i, (T, Hh) in enumerate(((Tq, Hq), (Tk, Hkv), (Tk, Hkv), (Tq, Hq))))
    want = R.attention(q, k, v, causal=causal, d_o=g)["dq"][0]
    leaves = [t.to(DEV).requires_grad_(True) for t in (q, k, v)]
    tokens.attention(*leaves, causal=causal).backward(g.to(DEV))
    off = lambda t: float((t.double().cpu() - want).norm() / want.norm())
    assert off(leaves[0].grad) < 1.25 * off(want.to(BF16)), (off(leaves[0].grad), off(want.to(BF16)))
