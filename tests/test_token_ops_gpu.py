"""GPU: the token operators (pdae_layernorm_*, pdae_dropout_*, pdae_mha_*) against their 64-bit restatements (tests/token_ref.py) at the sizes,
strides, lengths and masks where such kernels go wrong; the bounds are per element and count roundings."""
import math

import pytest
import torch

from tests import token_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF16 = torch.float32, torch.bfloat16


@pytest.fixture(scope="module")
def H():
    from pdae_amd import hip
    return hip


def rn(seed, *shape, dtype=F32, scale=1.0, shift=0.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale + shift).to(dtype)


def ws_of(nbytes, fill=float("nan")):
    return torch.full((max(4, (nbytes + 3) // 4),), fill, device=DEV)


def offset_copy(t, off):
    """A device copy of t that starts `off` elements behind an aligned address."""
    buf = torch.empty(t.numel() + off + 16, dtype=t.dtype, device=DEV)
    v = buf[off:off + t.numel()].view(t.shape)
    v.copy_(t)
    return v


# ------------------------------------------------------------------------------------------------ layer norm
LN = [(1, 1), (70, 64), (1100, 71), (37, 130), (2100, 128), (50, 250), (1500, 300), (1, 7000), (3, 2), (5, 7), (2, 8), (9, 63), (4, 65), (17, 512), (33, 520), (128, 2048), (6, 1000), (1030, 96), (4100, 40), (5, 2049), (3, 4099), (7, 8192), (2, 16384),
      (3, 16391), (2, 40000)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,C", LN)
def test_layernorm(H, rows, C, dtype):
    x, dy, add = rn(1, rows, C, dtype=dtype, scale=1.5, shift=0.5), rn(2, rows, C, dtype=dtype), rn(3, rows, C, dtype=dtype)
    gamma, beta = rn(4, C, scale=0.3, shift=1.0), rn(5, C)
    ref = R.layer_norm(x, gamma, beta, 1e-5, dy, add)
    k = H.DTYPES[dtype]
    xd, dyd, addd, gd, bd = (t.to(DEV) for t in (x, dy, add, gamma, beta))
    y, mean, rstd = torch.full_like(xd, float("nan")), torch.empty(rows, device=DEV), torch.empty(rows, device=DEV)
    H.run(H.op_layernorm_fwd(xd, gd, bd, rows, C, 1e-5, y, mean, rstd, dtype=k))
    for n, t in (("y", y), ("mean", mean), ("rstd", rstd)):
        R.within(t, ref[n], n)
    outs = []
    for _ in range(2):
        dx, dg, db = torch.full_like(xd, float("nan")), torch.full((C,), float("nan"), device=DEV), torch.full((C,), float("nan"), device=DEV)
        ws = ws_of(H.layernorm_ws_bytes(rows, C))
        H.run(H.op_layernorm_bwd(xd, gd, mean, rstd, dyd, rows, C, dx, dg, db, ws, add=addd, dtype=k))
        outs.append((dx, dg, db))
    for n, t in zip(("dx", "dgamma", "dbeta"), outs[0]):
        R.within(t, ref[n], n)
    assert all(torch.equal(a, b) for a, b in zip(*outs))                 # fixed summation order
    # "+=" into the weight gradients; dx over `add`
    dg, db = outs[0][1].clone(), outs[0][2].clone()
    H.run(H.op_layernorm_bwd(xd, gd, mean, rstd, dyd, rows, C, addd, dg, db, ws, add=addd, acc_param=1, dtype=k))
    assert torch.equal(addd, outs[0][0]) and torch.equal(dg, outs[0][1] * 2) and torch.equal(db, outs[0][2] * 2)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,C", [(1024, 130), (1025, 130), (1025, 9), (1030, 520), (1030, 1000), (1026, 1500), (1030, 2043), (1027, 4099), (1025, 8192)])
def test_layernorm_partial_rows(H, rows, C, dtype):
    """Around 1024 rows: below, blocks of columns add up the weight gradients in the same launch; above, the row blocks leave partial rows for a second one."""
    test_layernorm(H, rows, C, dtype)


def test_layernorm_more_rows_than_one_launch_holds(H):
    """2^22 blocks of 32 rows and five more rows; the statistics and rows around the seam and at the end."""
    rows, C = (32 << 22) + 5, 2
    x = torch.randn(rows, C, device=DEV, dtype=BF16)
    y, mean = torch.full_like(x, float("nan")), torch.full((rows,), float("nan"), device=DEV)
    H.run(H.op_layernorm_fwd(x, None, None, rows, C, 1e-5, y, mean, dtype=H.DT_BF16))
    for at in (0, rows - 37):
        ref = R.layer_norm(x[at:at + 37].cpu(), None, None, 1e-5)
        R.within(y[at:at + 37], ref["y"], "y"); R.within(mean[at:at + 37], ref["mean"], "mean")
    assert bool(torch.isfinite(mean).all())


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_layernorm_strides_offsets_and_optional_arguments(H, dtype):
    rows, C, ld = 37, 203, 260
    k = H.DTYPES[dtype]
    x, dy = rn(1, rows, C, dtype=dtype), rn(2, rows, C, dtype=dtype)
    ref = R.layer_norm(x, None, None, 1e-6, dy)

    def strided(t, off):
        buf = torch.full((rows * ld + off,), float("nan"), dtype=dtype, device=DEV)
        v = buf[off:].view(rows, ld)[:, :C]
        if t is not None:
            v.copy_(t)
        return v, buf
    (xv, _), (yv, yb), (dyv, _), (dxv, dxb) = strided(x, 1), strided(None, 3), strided(dy, 5), strided(None, 7)
    mean, rstd = torch.empty(rows, device=DEV), torch.empty(rows, device=DEV)
    H.run(H.op_layernorm_fwd(xv, None, None, rows, C, 1e-6, yv, mean, rstd, dtype=k, ldx=ld, ldy=ld))
    H.run(H.op_layernorm_bwd(xv, None, mean, rstd, dyv, rows, C, dxv, dtype=k, ldx=ld, lddy=ld, lddx=ld))
    R.within(yv, ref["y"], "y"); R.within(dxv, ref["dx"], "dx")
    assert int(torch.isfinite(yb).sum()) == rows * C and int(torch.isfinite(dxb).sum()) == rows * C      # nothing beside the rows was written
    y2 = torch.empty(rows, C, dtype=dtype, device=DEV)
    H.run(H.op_layernorm_fwd(xv, None, None, rows, C, 1e-6, y2, dtype=k, ldx=ld))                          # no statistics asked for
    assert torch.equal(y2, yv)
    dg = torch.empty(C, device=DEV)                                                                          # one of the two weight gradients
    H.run(H.op_layernorm_bwd(xv, None, mean, rstd, dyv, rows, C, dxv, dg, None, ws_of(H.layernorm_ws_bytes(rows, C)), dtype=k, ldx=ld, lddy=ld, lddx=ld))
    R.within(dg, ref["dgamma"], "dgamma")


def test_layernorm_large_mean_constant_rows_and_no_rows(H):
    """A mean 1000 times the deviation (E[x^2] - E[x]^2 would lose every digit), a constant row (variance 0), R = 0."""
    rows, C = 4, 1000
    x = rn(1, rows, C, scale=1.0, shift=1000.0)
    x[2] = 3.25
    ref = R.layer_norm(x, None, None, 1e-5)
    xd, y = x.to(DEV), torch.empty(rows, C, device=DEV)
    H.run(H.op_layernorm_fwd(xd, None, None, rows, C, 1e-5, y))
    R.within(y, ref["y"], "y")
    assert not y[2].any()
    dg = torch.full((C,), 7.0, device=DEV)
    H.run(H.op_layernorm_fwd(None, None, None, 0, C, 1e-5, None))
    H.run(H.op_layernorm_bwd(None, None, None, None, None, 0, C, None, dg, None, None, acc_param=1))
    assert bool((dg == 7).all())
    H.run(H.op_layernorm_bwd(None, None, None, None, None, 0, C, None, dg, None, None))
    assert not dg.any()


def test_layernorm_gradient_against_differences(H):
    """d/dx of sum(y * c) by central differences of the 64-bit forward agrees with the kernel's dx (fp32)."""
    rows, C = 3, 21
    x, dy, g, b = rn(1, rows, C), rn(2, rows, C), rn(3, C, shift=1.0), rn(4, C)
    xd = x.to(DEV)
    y, mean, rstd, dx = torch.empty_like(xd), torch.empty(rows, device=DEV), torch.empty(rows, device=DEV), torch.empty_like(xd)
    H.run(H.op_layernorm_fwd(xd, g.to(DEV), b.to(DEV), rows, C, 1e-5, y, mean, rstd))
    H.run(H.op_layernorm_bwd(xd, g.to(DEV), mean, rstd, dy.to(DEV), rows, C, dx))

    def f(t):
        m = t.mean(1, keepdim=True)
        return ((t - m) / ((t - m) ** 2).mean(1, keepdim=True).add(1e-5).sqrt() * g.double() + b.double()).mul(dy.double()).sum()
    eps, num = 1e-5, torch.zeros(rows, C, dtype=torch.double)
    for i in range(rows):
        for j in range(C):
            e = torch.zeros(rows, C, dtype=torch.double)
            e[i, j] = eps
            num[i, j] = (f(x.double() + e) - f(x.double() - e)) / (2 * eps)
    assert float((dx.double().cpu() - num).abs().max()) < 1e-5 * float(num.abs().max())


# ------------------------------------------------------------------------------------------------ dropout
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n", [1, 3, 7, 8, 9, 4096, 10001, 3000017])
def test_dropout(H, n, dtype):
    p, seed, step, layer = 0.3, 0x1234567890ABCD, 77, 5
    keep = R.keep_mask(n, p, seed, step, layer)
    x, res, k = rn(1, n, dtype=dtype), rn(2, n, dtype=dtype), H.DTYPES[dtype]
    u = R.U[dtype]
    d = torch.where(keep, x.double() / (1 - p), 0.0)
    for off in (0, 1):
        xd, rd = offset_copy(x, off), offset_copy(res, 2 * off)
        y = offset_copy(torch.full((n,), float("nan"), dtype=dtype), off)
        H.run(H.op_dropout_fwd(xd, rd, n, p, y, seed=seed, offset=step, layer=layer, dtype=k))
        want = d + res.double()
        R.within(y, (want, u * want.abs() + 4 * R.F * (d.abs() + want.abs())), "y")
        H.run(H.op_dropout_fwd(xd, None, n, p, y, seed=seed, offset=step, layer=layer, dtype=k))
        R.within(y, (d, u * d.abs() + 4 * R.F * d.abs()), "y without residual")
        assert torch.equal(y.cpu() != 0, keep & (x != 0))
        dx = offset_copy(res, off)
        H.run(H.op_dropout_bwd(xd, n, p, dx, seed=seed, offset=step, layer=layer, dtype=k))
        assert torch.equal(dx, y)                                          # the same mask from the same counter
        dx = offset_copy(res, off)
        H.run(H.op_dropout_bwd(xd, n, p, dx, seed=seed, offset=step, layer=layer, acc=1, dtype=k))
        R.within(dx, (want, u * want.abs() + 4 * R.F * (d.abs() + want.abs())), "dx +=")


def test_dropout_in_place_non_finite_and_p_zero(H):
    n, p = 1000, 0.5
    keep = R.keep_mask(n, p, 3, 4)
    x = rn(1, n)
    x[~keep] = float("inf")                                                # a dropped infinity is a zero, not a NaN
    x[int((~keep).nonzero()[0])] = float("nan")
    xd = x.to(DEV)
    H.run(H.op_dropout_fwd(xd, None, n, p, xd, seed=3, offset=4))
    assert torch.equal(xd.cpu(), torch.where(keep, x * 2, torch.zeros(())))
    y = torch.empty(n, device=DEV)
    H.run(H.op_dropout_fwd(x.to(DEV), None, n, 0.0, y, seed=3, offset=4))
    assert torch.equal(torch.nan_to_num(y.cpu(), nan=9.0), torch.nan_to_num(x, nan=9.0))
    H.run(H.op_dropout_fwd(None, None, 0, p, None))


def test_dropout_is_the_group_norm_kernels_mask_and_layers_differ(H):
    """The same (p, seed, step) drops the same elements as pdae_gn_apply; the layer number gives independent streams."""
    N, S, C, p = 2, 16, 64, 0.25
    n = N * S * S * C
    x = torch.ones(N, S, S, C, device=DEV)
    coef = torch.zeros(3, N, C, device=DEV)
    coef[1] = 1.0
    y = torch.empty_like(x)
    H.run(H.op_gn_apply(x, C, None, 0, N, S, S, coef, 0, 0, y, drop_p=p, seed=99, offset=5))
    z = torch.empty_like(x)
    H.run(H.op_dropout_fwd(x, None, n, p, z, seed=99, offset=5))
    assert torch.equal(y != 0, z != 0)
    masks = []
    for layer in (1, 2):
        H.run(H.op_dropout_fwd(x, None, n, p, z, seed=99, offset=5, layer=layer))
        masks.append((z != 0).float().flatten())
    for m in masks:
        assert abs(float(m.mean()) - (1 - p)) < 6 * math.sqrt(p * (1 - p) / n)
    agree = float((masks[0] == masks[1]).float().mean())
    assert abs(agree - (p * p + (1 - p) ** 2)) < 6 * math.sqrt(0.25 / n)


# ------------------------------------------------------------------------------------------------ attention
def run_mha(H, q, k, v, d_o=None, q_len=None, k_len=None, causal=False, scale=None, layout="plain", fill=float("nan")):
    """Runs the kernels on copies in the given layout; outputs start as NaN (every element has to be written)."""
    B, Tq, Hq, D = q.shape
    Tk, Hkv = k.shape[1], k.shape[2]
    dt = q.dtype

    def place(t):
        B_, T_, H_, D_ = t.shape
        if layout == "plain":
            return t.to(DEV).contiguous()
        if layout == "heads":                                                # [batch][head][token][channel]
            return t.permute(0, 2, 1, 3).contiguous().to(DEV).permute(0, 2, 1, 3)
        buf = torch.full((B_ * T_ * H_ * (D_ + 3) + 5,), fill, dtype=dt, device=DEV)        # odd row length, odd start
        w = buf[5:].view(B_, T_, H_, D_ + 3)[..., :D_]
        w.copy_(t)
        return w
    qd, kd, vd = place(q), place(k), place(v)
    ob = place(torch.full_like(q, fill))
    ln = [None if t is None else torch.tensor(t, dtype=torch.int32, device=DEV) for t in (q_len, k_len)]
    a = H.Mha(B, Tq, Tk, Hq, Hkv, D, dtype=H.DTYPES[dt], causal=causal, scale=scale, q_stride=qd.stride()[:3], k_stride=kd.stride()[:3], v_stride=vd.stride()[:3],
              o_stride=ob.stride()[:3])
    lse = torch.full((B, Hq, Tq), fill, device=DEV)
    ws = ws_of(a.ws_bytes(d_o is not None))
    H.run(H.op_mha_fwd(a, qd, kd, vd, ob, lse=lse, q_len=ln[0], k_len=ln[1], ws=ws))
    got = dict(o=ob, lse=lse)
    o2 = place(torch.full_like(q, fill))
    H.run(H.op_mha_fwd(a, qd, kd, vd, o2, q_len=ln[0], k_len=ln[1], ws=ws))                 # without lse
    assert torch.equal(o2, ob)
    if d_o is not None:
        runs = []
        for _ in range(2):
            g = place(d_o)
            dq, dk, dv = place(torch.full_like(q, fill)), place(torch.full_like(k, fill)), place(torch.full_like(v, fill))
            ws.fill_(fill)
            H.run(H.op_mha_bwd(a, qd, kd, vd, ob, lse, g, dq, dk, dv, q_len=ln[0], k_len=ln[1], ws=ws))
            runs.append((dq, dk, dv))
        assert all(torch.equal(x, y) for x, y in zip(*runs))
        got.update(zip(("dq", "dk", "dv"), runs[0]))
    return got


def check_mha(H, B, Tq, Tk, Hq, Hkv, D, dtype, causal=False, q_len=None, k_len=None, scale=None, layout="plain", spread=1.0, junk=False):
    q, k, v = rn(1, B, Tq, Hq, D, dtype=dtype, scale=spread), rn(2, B, Tk, Hkv, D, dtype=dtype, scale=spread), rn(3, B, Tk, Hkv, D, dtype=dtype)
    g = rn(4, B, Tq, Hq, D, dtype=dtype)
    ref = R.attention(q, k, v, q_len, k_len, causal, scale, g)
    if junk:                                                                 # NaN and infinities where nothing may be read
        for b in range(B):
            lq, lk = q_len[b], k_len[b]
            for t, n in ((q, lq), (g, lq), (k, lk), (v, lk)):
                t[b, n:] = float("nan")
                t[b, n + 1::2] = float("inf")
    got = run_mha(H, q, k, v, g, q_len, k_len, causal, scale, layout)
    for n in ("o", "lse", "dq", "dk", "dv"):
        R.within(got[n], ref[n], n)


SHAPES = [(1, 1, 1, 1, 1, 1), (2, 1, 33, 4, 2, 64), (1, 3, 257, 6, 1, 40), (2, 64, 64, 2, 2, 32), (1, 65, 63, 2, 1, 33), (2, 129, 200, 3, 3, 72), (1, 128, 128, 4, 4, 64),
          (1, 257, 300, 4, 2, 128), (3, 31, 513, 2, 2, 96), (1, 300, 31, 2, 1, 80), (1, 1, 2100, 8, 2, 128), (2, 5, 1500, 4, 4, 24), (1, 190, 190, 1, 1, 127)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_attention_forward_backward(H, shape, causal, dtype):
    check_mha(H, *shape, dtype, causal)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("D", [64, 100, 128])
def test_attention_padded_batch(H, D, causal, dtype):
    """Lengths 0, 1, full and in between, on both sides; whatever lies behind them (NaN, infinities) is not read, and comes out as zero."""
    check_mha(H, 6, 150, 170, 4, 2, D, dtype, causal, q_len=[150, 0, 1, 149, 33, 64], k_len=[170, 5, 0, 1, 65, 128], junk=True)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("layout", ["heads", "odd"])
def test_attention_strides(H, layout, dtype):
    check_mha(H, 2, 70, 90, 4, 2, 48, dtype, True, layout=layout)
    check_mha(H, 2, 70, 90, 4, 2, 47, dtype, False, q_len=[70, 3], k_len=[2, 90], layout=layout)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_scales_and_large_scores(H, dtype):
    check_mha(H, 1, 80, 100, 2, 2, 64, dtype, scale=0.7)
    check_mha(H, 1, 80, 100, 2, 2, 64, dtype, True, scale=1e-4)
    # scores of a few hundred: the running maximum has to carry them
    q, k, v = rn(1, 1, 70, 2, 32, dtype=dtype, scale=8.0), rn(2, 1, 200, 2, 32, dtype=dtype, scale=8.0), rn(3, 1, 200, 2, 32, dtype=dtype)
    ref, got = R.attention(q, k, v), run_mha(H, q, k, v)
    R.within(got["o"], ref["o"], "o"); R.within(got["lse"], ref["lse"], "lse")


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_split_backward_and_long_rows(H, dtype):
    """Few heads and long rows: every kernel splits its summed axis and joins the partial results."""
    a = H.Mha(1, 1100, 900, 1, 1, 64, dtype=H.DTYPES[dtype])
    assert a.ws_bytes(True) > 4 * 1100 * 64                                    # partial results are there
    check_mha(H, 1, 1100, 900, 1, 1, 64, dtype)
    check_mha(H, 1, 300, 2100, 2, 1, 128, dtype, True, q_len=[299], k_len=[2050])


def test_attention_empty_axes(H):
    """No keys at all: every row is empty.  No queries: the key gradients are zero.  No samples: nothing happens."""
    for Tq, Tk, B in ((5, 0, 2), (0, 5, 2), (3, 3, 0)):
        q, k = torch.randn(B, Tq, 2, 16, device=DEV), torch.randn(B, Tk, 2, 16, device=DEV)
        o, dq, dk, dv = torch.full_like(q, 7.0), torch.full_like(q, 7.0), torch.full_like(k, 7.0), torch.full_like(k, 7.0)
        lse = torch.zeros(B, 2, Tq, device=DEV)
        a = H.Mha(B, Tq, Tk, 2, 2, 16)
        ws = ws_of(a.ws_bytes(True))
        H.run(H.op_mha_fwd(a, q, k, k, o, lse=lse, ws=ws))
        H.run(H.op_mha_bwd(a, q, k, k, o, lse, q, dq, dk, dv, ws=ws))
        for t in (o, dq, dk, dv):
            assert not t.any()
        assert bool((lse == -math.inf).all())


def test_attention_lengths_outside_the_tensor_are_cut(H):
    q, k, v, g = (rn(s, 2, 40, 2, 32).to(DEV) for s in (1, 2, 3, 4))
    a = H.Mha(2, 40, 40, 2, 2, 32)
    res = []
    for lens in ([40, 0], [10 ** 9, -5]):
        ln = torch.tensor(lens, dtype=torch.int32, device=DEV)
        o, lse, dq, dk, dv = torch.empty_like(q), torch.empty(2, 2, 40, device=DEV), torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
        ws = ws_of(a.ws_bytes(True))
        H.run(H.op_mha_fwd(a, q, k, v, o, lse=lse, q_len=ln, k_len=ln, ws=ws))
        H.run(H.op_mha_bwd(a, q, k, v, o, lse, g, dq, dk, dv, q_len=ln, k_len=ln, ws=ws))
        res.append((o, lse, dq, dk, dv))
    assert all(torch.equal(x, y) for x, y in zip(*res))


@pytest.mark.parametrize("lengths", [False, True])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("shape", [(128, 150, 140, 2, 2, 64), (64, 257, 100, 4, 2, 32), (43, 300, 70, 3, 1, 40), (256, 129, 65, 1, 1, 8), (64, 130, 700, 4, 4, 64)], ids=lambda s: "x".join(map(str, s)))
def test_attention_that_fills_the_chip(H, shape, causal, lengths):
    """Enough workgroups for 64 query rows a wave (bf16, D <= 64, more than 128 rows)."""
    B, Tq, Tk = shape[:3]
    ln = dict(q_len=[(37 * b) % (Tq + 1) for b in range(B)], k_len=[(53 * b) % (Tk + 1) for b in range(B)]) if lengths else {}
    check_mha(H, *shape, BF16, causal=causal, junk=lengths, **ln)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("Tq", [1, 150])
def test_attention_offsets_beyond_32_bits(H, Tq, dtype):
    """Keys 2^20 elements apart: offsets pass 2^31 elements inside one sample's cache.  The same bits as from a dense copy."""
    Tk, Hq, Hkv, D, st = 2100, 4, 2, 64, 1 << 20
    q, g = rn(1, 1, Tq, Hq, D, dtype=dtype).to(DEV), rn(2, 1, Tq, Hq, D, dtype=dtype).to(DEV)
    kv = rn(3, 2, 1, Tk, Hkv, D, dtype=dtype).to(DEV)
    wide = lambda: torch.empty(Tk * st, dtype=dtype, device=DEV).as_strided((1, Tk, Hkv, D), (Tk * st, st, D, 1))
    outs = []
    for far in (False, True):
        k, dk = (wide(), wide()) if far else (torch.empty(1, Tk, Hkv, D, dtype=dtype, device=DEV) for _ in range(2))
        v, dv = (t.as_strided(t.shape, t.stride(), 4096) if far else torch.empty_like(t) for t in (k, dk))     # v lies in the gaps of k
        k.copy_(kv[0]); v.copy_(kv[1])
        a = H.Mha(1, Tq, Tk, Hq, Hkv, D, dtype=H.DTYPES[dtype], causal=True, k_stride=k.stride()[:3], v_stride=v.stride()[:3])
        o, dq, lse, ws = torch.empty_like(q), torch.empty_like(q), torch.empty(1, Hq, Tq, device=DEV), ws_of(a.ws_bytes(True))
        H.run(H.op_mha_fwd(a, q, k, v, o, lse=lse, ws=ws))
        H.run(H.op_mha_bwd(a, q, k, v, o, lse, g, dq, dk, dv, ws=ws))
        outs.append([t.contiguous().clone() for t in (o, lse, dq, dk, dv)])
        assert torch.equal(k, kv[0]) and torch.equal(v, kv[1])
    assert all(torch.equal(x, y) for x, y in zip(*outs))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("Tq", [3, 200])
def test_attention_keeps_a_bad_row_to_itself_and_shows_a_bad_key(H, Tq, dtype):
    """NaN in a query makes that row NaN and no other; NaN in a visible key or value reaches every row that sees it."""
    q, k, v = rn(1, 1, Tq, 2, 64, dtype=dtype), rn(2, 1, 300, 2, 64, dtype=dtype), rn(3, 1, 300, 2, 64, dtype=dtype)
    ref = R.attention(q, k, v)
    a = H.Mha(1, Tq, 300, 2, 2, 64, dtype=H.DTYPES[dtype])

    def run(q, k, v):
        o = torch.empty(q.shape, dtype=dtype, device=DEV)
        H.run(H.op_mha_fwd(a, q.to(DEV), k.to(DEV), v.to(DEV), o, ws=ws_of(a.ws_bytes())))
        return o.cpu()
    bad = q.clone()
    bad[0, 1, 0, 5] = float("nan")
    o = run(bad, k, v)
    assert bool(torch.isnan(o[0, 1, 0]).all())
    o[0, 1, 0] = ref["o"][0][0, 1, 0].to(dtype)
    R.within(o, ref["o"], "o")
    for t in (k, v):
        bad = t.clone()
        bad[0, 299, 1] = float("nan")
        o = run(q, *((bad, v) if t is k else (k, bad)))
        assert bool(torch.isnan(o[:, :, 1]).all())
        R.within(o[:, :, :1], tuple(x[:, :, :1] for x in ref["o"]), "o")


def test_attention_agrees_with_the_fused_image_attention(H):
    """The same qkv tensor through pdae_attn_fwd / _bwd (64 .. 256 tokens) and through the general kernels by strides, both channel orders."""
    N, T, C, heads = 2, 64, 128, 2
    ch = C // heads
    qkv, g = rn(1, N, T, 3 * C).to(DEV), rn(2, N, T, C).to(DEV)
    for order in (False, True):
        oq, ok, ov, hs = (0, C, 2 * C, ch) if order else (0, ch, 2 * ch, 3 * ch)
        out, lse = torch.empty(N, T, C, device=DEV), torch.empty(N * heads, T, device=DEV)
        H.run(H.op_attn_fwd(qkv, N, T, C, heads, order, out, lse))
        d1 = torch.empty_like(qkv)
        H.run(H.op_attn_bwd(qkv, out, lse, g, N, T, C, heads, order, d1, torch.empty(N * heads, T, device=DEV)))
        st = (T * 3 * C, 3 * C, hs)
        a = H.Mha(N, T, T, heads, heads, ch, q_stride=st, k_stride=st, v_stride=st, o_stride=(T * C, C, ch))
        o2, l2, d2 = torch.empty_like(out), torch.empty_like(lse), torch.full_like(qkv, float("nan"))
        p, dp = qkv.data_ptr(), d2.data_ptr()
        ws = ws_of(a.ws_bytes(True))
        H.run(H.op_mha_fwd(a, p + 4 * oq, p + 4 * ok, p + 4 * ov, o2, lse=l2, ws=ws))
        H.run(H.op_mha_bwd(a, p + 4 * oq, p + 4 * ok, p + 4 * ov, o2, l2, g, dp + 4 * oq, dp + 4 * ok, dp + 4 * ov, ws=ws))
        for x, y in ((out, o2), (lse, l2), (d1, d2)):
            assert float((x - y).abs().max()) < 1e-5 * float(x.abs().max())


def test_attention_gradient_against_differences(H):
    """Directional derivative of sum(o * g) along a random direction of (q, k, v): kernel gradients against central differences in 64 bits."""
    B, T, Hh, D = 1, 37, 2, 24
    q, k, v, g = (rn(s, B, T, Hh, D) for s in (1, 2, 3, 4))
    dirs = [rn(s, B, T, Hh, D).double() for s in (5, 6, 7)]
    got = run_mha(H, q, k, v, g, causal=True)

    def f(e):
        qq, kk, vv = (t.double() + e * d for t, d in zip((q, k, v), dirs))
        s = torch.einsum("bihd,bjhd->bhij", qq, kk) / math.sqrt(D)
        s = s.masked_fill(torch.ones(T, T, dtype=torch.bool).triu(1), -math.inf)
        return float((torch.einsum("bhij,bjhd->bihd", torch.softmax(s, -1), vv) * g.double()).sum())
    num = (f(1e-5) - f(-1e-5)) / 2e-5
    ana = sum(float((got[n].double().cpu() * d).sum()) for n, d in zip(("dq", "dk", "dv"), dirs))
    assert abs(num - ana) < 1e-5 * max(1.0, abs(num))
