"""CPU: what the token operators refuse, their record layouts and workspace sizes, and the 64-bit restatements the GPU tests use."""
import ctypes
import math

import pytest
import torch

from tests import token_ref as R


@pytest.fixture(scope="module")
def H():
    from pdae_amd.build import build_library
    build_library(verbose=False)
    from pdae_amd import hip
    return hip


def refuses(H, op, match):
    with pytest.raises(H.PdaeError, match=match):
        H.run(op, stream=0)


P = 4096        # stands for a device pointer: every call here ends before a launch


def test_layernorm_refusals(H):
    ok = dict(dtype=H.DT_F32)
    refuses(H, H.op_layernorm_fwd(P, P, P, 4, 0, 1e-5, P, **ok), "C > 0")
    refuses(H, H.op_layernorm_fwd(P, P, P, -1, 8, 1e-5, P, **ok), "R >= 0")
    refuses(H, H.op_layernorm_fwd(P, P, P, 4, 8, -1.0, P, **ok), "eps")
    refuses(H, H.op_layernorm_fwd(P, P, P, 4, 8, float("nan"), P, **ok), "eps")
    refuses(H, H.op_layernorm_fwd(None, P, P, 4, 8, 1e-5, P, **ok), "null")
    refuses(H, H.op_layernorm_fwd(P, P, P, 4, 8, 1e-5, P, dtype=2), "dtype")
    refuses(H, H.op_layernorm_fwd(P, P, P, 4, 8, 1e-5, P, ldx=7, **ok), "stride")
    refuses(H, H.op_layernorm_fwd(P + 2, P, P, 4, 8, 1e-5, P, **ok), "aligned")
    bwd = lambda ws, n, **k: H.op_layernorm_bwd(P, P, P, P, P, 4, 8, P, P, P, ws, ws_bytes=n, **k)
    refuses(H, bwd(None, 0), "workspace")
    refuses(H, bwd(P, H.layernorm_ws_bytes(4, 8) - 1), "workspace")
    refuses(H, bwd(P, 1 << 20, lddx=4), "stride")
    refuses(H, H.op_layernorm_bwd(P, P, None, P, P, 4, 8, P), "null")


def test_dropout_refusals(H):
    for p in (-0.1, 1.0, 1.5, float("nan")):
        refuses(H, H.op_dropout_fwd(P, None, 8, p, P), r"\[0, 1\)")
    refuses(H, H.op_dropout_fwd(P, None, -8, 0.1, P), "negative")
    refuses(H, H.op_dropout_fwd(None, None, 8, 0.1, P), "null")
    refuses(H, H.op_dropout_fwd(P, None, 8, 0.1, P, dtype=7), "dtype")
    refuses(H, H.op_dropout_bwd(P, 8, 0.1, P + 1, dtype=H.DT_BF16), "aligned")


def test_attention_refusals(H):
    def fwd(a, q=P, k=P, v=P, o=P, **kw):
        return H.op_mha_fwd(a, q, k, v, o, **kw)
    good = dict(B=2, Tq=4, Tk=4, Hq=2, Hkv=1, D=8)
    refuses(H, fwd(H.Mha(**dict(good, D=129))), "head width")
    refuses(H, fwd(H.Mha(**dict(good, D=0), scale=1.0)), "head width")
    refuses(H, fwd(H.Mha(**dict(good, Hq=3, Hkv=2))), "share")
    refuses(H, fwd(H.Mha(**dict(good, Tq=-1))), "bad sizes")
    refuses(H, fwd(H.Mha(**good, dtype=3)), "dtype")
    for s in (0.0, -1.0, float("inf"), float("nan")):
        refuses(H, fwd(H.Mha(**good, scale=s)), "scale")
    refuses(H, fwd(H.Mha(**good), q=None), "null")
    refuses(H, fwd(H.Mha(**good), k=None), "null")
    refuses(H, fwd(H.Mha(**good, dtype=H.DT_BF16), v=P + 1), "aligned")
    refuses(H, fwd(H.Mha(**good, k_stride=(-1, 8, 8))), "stride")
    refuses(H, fwd(H.Mha(**good, o_stride=(64, 8, 8))), "rows of o overlap")
    refuses(H, fwd(H.Mha(**good, o_stride=(64, 16, 4))), "rows of o overlap")
    a = H.Mha(1, 1, 4096, 2, 1, 64)
    assert a.ws_bytes() > 0
    refuses(H, fwd(a), "workspace")
    refuses(H, fwd(a, ws=P, ws_bytes=a.ws_bytes() - 1), "workspace")

    def bwd(a, **kw):
        base = dict(q=P, k=P, v=P, o=P, lse=P, d_o=P, dq=P, dk=P, dv=P, ws=P, ws_bytes=1 << 40)
        return H.op_mha_bwd(a, **dict(base, **kw))
    refuses(H, bwd(H.Mha(**good), lse=None), "null")
    refuses(H, bwd(H.Mha(**good), dv=None), "null")
    refuses(H, bwd(H.Mha(**good), ws=None, ws_bytes=0), "workspace")
    # a key head that is broadcast over the batch by a zero stride can be read, its gradient has no place
    refuses(H, bwd(H.Mha(**good, k_stride=(0, 8, 8))), "rows of dk")
    refuses(H, bwd(H.Mha(**good, v_stride=(0, 8, 8))), "rows of dv")
    refuses(H, bwd(H.Mha(**good, q_stride=(0, 16, 8))), "rows of dq")


def test_sizes_and_strides_beyond_the_kernels_are_refused(H):
    good = dict(B=2, Tq=4, Tk=4, Hq=2, Hkv=1, D=8)
    fwd = lambda a: H.op_mha_fwd(a, P, P, P, P)
    refuses(H, fwd(H.Mha(**good, v_stride=(1 << 30, 1 << 21, 8))), "token stride")
    refuses(H, fwd(H.Mha(**good, q_stride=(1 << 39, 16, 1 << 30))), "head stride")                # two heads are rows of one tile
    refuses(H, fwd(H.Mha(**dict(good, B=1 << 20), k_stride=(1 << 39, 8, 8))), "beyond every address")
    refuses(H, fwd(H.Mha(**dict(good, B=1 << 25, Hq=1))), "too many query rows")
    refuses(H, H.op_mha_bwd(H.Mha(**dict(good, B=1 << 25, Hq=1)), P, P, P, P, P, P, P, P, P, ws=P, ws_bytes=1 << 60), "too many")
    refuses(H, fwd(H.Mha(**dict(good, Tq=(1 << 32) + 4))), r"2\^31")                               # (4 if it were cut to 32 bits)
    refuses(H, H.op_layernorm_fwd(P, P, P, (1 << 32) + 4, 8, 1e-5, P), r"2\^31")
    refuses(H, H.op_layernorm_bwd(P, P, P, P, P, 4, (1 << 32) + 8, P), r"2\^31")
    refuses(H, H.op_layernorm_fwd(P, P, P, 4, (1 << 24) + 1, 1e-5, P), r"2\^24")
    refuses(H, H.op_layernorm_bwd(P, P, P, P, P, 4, 8, P, P, P, P + 2, ws_bytes=1 << 20), "aligned")


def test_token_functions_refuse(H):
    import torch
    from pdae_amd import tokens
    x = torch.zeros(2, 8)
    for f in (lambda: tokens.layer_norm(x), lambda: tokens.dropout(x, 0.1, 0), lambda: tokens.attention(*(torch.zeros(1, 2, 1, 8),) * 3)):
        with pytest.raises(H.PdaeError, match="no CPU fallback"):
            f()
    for k in (dict(step=1 << 32), dict(step=-1), dict(layer=1 << 32)):
        with pytest.raises(H.PdaeError, match="must lie in"):
            tokens.dropout(x, 0.1, 0, **k)
    row = torch.zeros(1, 9, 2, 8)
    assert tokens._own_rows(row) and tokens._own_rows(row.transpose(1, 2)) and not tokens._own_rows(row.expand(3, 9, 2, 8))
    assert not tokens._own_rows(row.as_strided((1, 4, 2, 8), (144, 8, 16, 1)))                     # windows that share tokens


def test_refused_op_names_its_place(H):
    ops = H.ops_array([H.op_dropout_fwd(None, None, 0, 0.1, None), H.op_dropout_fwd(P, None, 8, 2.0, P)])
    with pytest.raises(H.PdaeError, match=r"op 1 \(kind %d\)" % H.OP_DROPOUT_FWD):
        H.run_ops(ops, 2, stream=0)


def test_struct_and_workspace_sizes(H):
    assert ctypes.sizeof(H.MhaDesc) == 8 * 4 + 12 * 8 + 8
    assert H.layernorm_ws_bytes(1, 10) == 2 * 10 * 4 and H.layernorm_ws_bytes(10 ** 6, 100) <= 1024 * 2 * 100 * 4
    assert H.Mha(64, 1024, 1024, 16, 16, 64).ws_bytes() == 0                  # enough tiles: nothing is split
    assert H.Mha(64, 1024, 1024, 16, 16, 64).ws_bytes(True) == 64 * 16 * 1024 * 4   # delta only
    assert H.Mha(0, 4, 4, 1, 1, 8).ws_bytes(True) == 0


def test_plan_check_knows_the_ops(H):
    from pdae_amd import plancheck
    for n in ("OP_LAYERNORM_FWD", "OP_LAYERNORM_BWD", "OP_DROPOUT_FWD", "OP_DROPOUT_BWD", "OP_MHA_FWD", "OP_MHA_BWD"):
        assert getattr(H, n) in plancheck.WRITES
    a = H.Mha(1, 2, 2, 1, 1, 8)
    r, w = plancheck.op_sets(H.op_mha_bwd(a, 1, 2, 3, 4, 5, 6, 7, 8, 9, q_len=10, k_len=11, ws=12), [])
    assert r == {1, 2, 3, 4, 5, 6, 10, 11} and w == {7, 8, 9, 12}


def test_restatements_agree_with_autograd():
    """The 64-bit restatements against torch's own differentiation of the same formulas."""
    g = torch.Generator().manual_seed(0)
    B, Tq, Tk, Hq, Hkv, D = 2, 7, 9, 4, 2, 5
    q, k, v, d_o = (torch.randn(B, T, Hh, D, generator=g) for T, Hh in ((Tq, Hq), (Tk, Hkv), (Tk, Hkv), (Tq, Hq)))
    ref = R.attention(q, k, v, [7, 4], [9, 2], True, None, d_o)
    Q, K, V = (t.double().requires_grad_(True) for t in (q, k, v))
    total = 0.0
    for b, (n, m) in enumerate(((7, 9), (4, 2))):
        for h in range(Hq):
            s = Q[b, :n, h] @ K[b, :m, h // 2].T / math.sqrt(D)
            s = s.masked_fill(torch.ones(n, m, dtype=torch.bool).triu(m - n + 1), -math.inf)[max(0, n - m):]
            o = torch.softmax(s, 1) @ V[b, :m, h // 2]
            total = total + (o * d_o[b, max(0, n - m):n, h].double()).sum()
    total.backward()
    for name, t in (("dq", Q), ("dk", K), ("dv", V)):
        assert float((ref[name][0] - t.grad).abs().max()) < 1e-12
    x, dy, gm, bt = torch.randn(3, 11, generator=g), torch.randn(3, 11, generator=g), torch.randn(11, generator=g), torch.randn(11, generator=g)
    X, G, Bt = x.double().requires_grad_(True), gm.double().requires_grad_(True), bt.double().requires_grad_(True)
    y = torch.nn.functional.layer_norm(X, (11,), G, Bt, 1e-5)
    (y * dy.double()).sum().backward()
    ln = R.layer_norm(x, gm, bt, 1e-5, dy)
    for n, t in (("y", y), ("dx", X.grad), ("dgamma", G.grad), ("dbeta", Bt.grad)):
        assert float((ln[n][0] - t.detach()).abs().max()) < 1e-12
    keep = R.keep_mask(1 << 16, 0.1, 5, 6)
    assert abs(float(keep.double().mean()) - 0.9) < 6 * math.sqrt(0.09 / (1 << 16))


def test_tensor_functions_have_no_cpu_fallback():
    from pdae_amd import tokens
    from pdae_amd.hip import PdaeError
    x = torch.zeros(2, 3, 1, 8)
    for call in (lambda: tokens.layer_norm(x), lambda: tokens.dropout(x, 0.1, 0), lambda: tokens.attention(x, x, x)):
        with pytest.raises(PdaeError, match="ROCm device"):
            call()


def test_latent_denoiser_plans_dropout():
    """MLPSkipNet's training plan drops behind every layer but the last, once per direction, with a stream per layer; evaluation and sampling plans do not."""
    from pdae_amd import hip as H
    from pdae_amd.model.mlp_skip_net import MLPSkipNet
    net = MLPSkipNet(input_channel=16, model_channel=32, num_layers=4, time_emb_channel=8, use_norm=True, dropout=0.1, device="cpu")
    kinds = lambda p: [(r.kind, r.i[4], round(r.f[0], 6)) for r in p.recs if r.kind in (H.OP_DROPOUT_FWD, H.OP_DROPOUT_BWD)]
    net.train()
    p = net.plan(4, True)
    assert kinds(p) == [(H.OP_DROPOUT_FWD, i, 0.1) for i in (1, 2, 3)] + [(H.OP_DROPOUT_BWD, i, 0.1) for i in (3, 2, 1)]
    p.set_dropout(12345, 6)
    assert all(p.arr[k].i[2] == 12345 and p.arr[k].i[3] == 6 for k, _, _ in p.drop_ops) and len(p.drop_ops) == 6
    assert not kinds(net.plan(4, False))
    net.eval()
    assert not kinds(net.plan(4, True))
    for bad in (1.0, -0.1):
        with pytest.raises(AssertionError):
            MLPSkipNet(input_channel=16, model_channel=32, num_layers=3, time_emb_channel=8, use_norm=True, dropout=bad, device="cpu")
