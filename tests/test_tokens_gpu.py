"""GPU: the token operators as a program uses them -- together in a block through the tensor-level functions (pdae_amd/tokens.py), inside planned networks
(MLPSkipNet's dropout, AttentionBlock at sizes the fused kernels do not take), captured into graphs, on other streams, two at a time."""
import math
import random

import pytest
import torch
import torch.nn.functional as F

from tests import token_ref as R
from tests.conftest import rel_err
from tests.golden import make_fixtures_cfg as C

pytestmark = pytest.mark.gpu
DEV = "cuda"


def rn(seed, *shape, scale=1.0, shift=0.0):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=g) * scale + shift


# ------------------------------------------------------------------------------------------------ together
def block(x, P, tok, heads, kv, p, mm=torch.matmul):
    """Pre-norm token block: x + drop(proj(attention(norm(x)))), then the same around a two-layer MLP.  tok: (layer_norm, attention, dropout)."""
    norm, attn, drop = tok
    B, T, W = x.shape
    D = W // heads
    h = norm(x, P["g1"], P["b1"])
    qkv = mm(h, P["qkv"])
    q = qkv[..., :W].view(B, T, heads, D)
    k = qkv[..., W:W + kv * D].view(B, T, kv, D)
    v = qkv[..., W + kv * D:].view(B, T, kv, D)
    o = attn(q, k, v).reshape(B, T, W)
    x = drop(mm(o, P["proj"]), p, 1, x)
    h = norm(x, P["g2"], P["b2"])
    return drop(mm(F.silu(mm(h, P["fc1"])), P["fc2"]), p, 2, x)


def block_params(W, heads, kv, seed=0):
    D = W // heads
    s = [rn(seed + i, *shape, scale=1 / math.sqrt(shape[0])) for i, shape in enumerate(((W, W + 2 * kv * D), (W, W), (W, 2 * W), (2 * W, W)))]
    return dict(qkv=s[0], proj=s[1], fc1=s[2], fc2=s[3], g1=rn(9, W, scale=0.2, shift=1.0), b1=rn(10, W, scale=0.1), g2=rn(11, W, scale=0.2, shift=1.0),
                b2=rn(12, W, scale=0.1))


def test_token_block_forward_and_gradients_against_64_bits():
    """All operators in one block with shared key heads, a ragged causal batch and dropout, fp32.  Bound: ten stages, each of at most K + 20 <= 150 fp32 roundings
    of its largest terms (150 x 2^-24 = 9e-6), gives 1e-4 of the largest value."""
    from pdae_amd import tokens
    B, T, W, heads, kv, p = 3, 37, 64, 4, 2, 0.2
    lens = [37, 20, 1]
    ln = torch.tensor(lens, dtype=torch.int32, device=DEV)
    x, dy = rn(1, B, T, W), rn(2, B, T, W)
    P = block_params(W, heads, kv)
    xd = x.to(DEV).requires_grad_(True)
    Pd = {k: v.to(DEV).requires_grad_(True) for k, v in P.items()}
    tok = (tokens.layer_norm, lambda q, k, v: tokens.attention(q, k, v, q_len=ln, k_len=ln, causal=True),
           lambda t, p, layer, res: tokens.dropout(t, p, 77, step=5, layer=layer, residual=res))
    y = block(xd, Pd, tok, heads, kv, p)
    y.backward(dy.to(DEV))

    def attn64(q, k, v):
        out = torch.zeros_like(q)
        for b, n in enumerate(lens):
            rows = []
            for h in range(heads):
                s = (q[b, :n, h] @ k[b, :n, h // 2].T / math.sqrt(W // heads)).masked_fill(torch.ones(n, n, dtype=torch.bool).triu(1), -math.inf)
                rows.append(torch.softmax(s, -1) @ v[b, :n, h // 2])
            out = torch.cat([out[:b], torch.cat([torch.stack(rows, 1), torch.zeros(T - n, heads, W // heads, dtype=q.dtype)])[None], out[b + 1:]])
        return out

    def drop64(t, p, layer, res):
        keep = R.keep_mask(t.numel(), p, 77, 5, layer).view_as(t)
        return res + torch.where(keep, t / (1 - p), torch.zeros_like(t))
    x6 = x.double().requires_grad_(True)
    P6 = {k: v.double().requires_grad_(True) for k, v in P.items()}
    y6 = block(x6, P6, (lambda t, g, b: F.layer_norm(t, (W,), g, b, 1e-5), attn64, drop64), heads, kv, p)
    y6.backward(dy.double())
    assert rel_err(y, y6.detach()) < 1e-4
    assert rel_err(xd.grad, x6.grad) < 1e-4
    for k in P:
        assert rel_err(Pd[k].grad, P6[k].grad) < 1e-4, k


def test_token_block_bf16_runs_and_repeats():
    """bf16 activations: finite outputs and gradients, and the same bits on a second run (no atomics anywhere)."""
    from pdae_amd import tokens
    B, T, W, heads, kv = 2, 300, 256, 4, 4
    P = {k: v.to(DEV) for k, v in block_params(W, heads, kv).items()}
    x, dy = rn(1, B, T, W).to(DEV).bfloat16(), rn(2, B, T, W).to(DEV).bfloat16()
    mm = lambda a, w: torch.mm(a.reshape(-1, a.shape[-1]), w.to(a.dtype)).view(*a.shape[:-1], w.shape[1])
    tok = (tokens.layer_norm, tokens.attention, lambda t, p, layer, res: tokens.dropout(t, p, 3, layer=layer, residual=res))
    runs = []
    for _ in range(2):
        xr = x.clone().requires_grad_(True)
        g1 = P["g1"].clone().requires_grad_(True)
        y = block(xr, dict(P, g1=g1), tok, heads, kv, 0.1, mm)
        y.backward(dy)
        runs.append((y.detach(), xr.grad, g1.grad))
    for a, b in zip(*runs):
        assert torch.isfinite(a.float()).all() and torch.equal(a, b)


# ------------------------------------------------------------------------------------------------ tensor-level functions
def test_functions_take_views_broadcasts_and_expanded_gradients():
    from pdae_amd import tokens
    # a strided 2-D view, an expanded output gradient (sum), no bias
    base = rn(1, 9, 100).to(DEV)
    x = base[:, 10:74].detach().requires_grad_(True)
    g = rn(2, 64, shift=1.0).to(DEV).requires_grad_(True)
    tokens.layer_norm(x, g).sum().backward()
    x6, g6 = base[:, 10:74].double().cpu().requires_grad_(True), g.detach().double().cpu().requires_grad_(True)
    F.layer_norm(x6, (64,), g6, None, 1e-5).sum().backward()
    assert float((x.grad.double().cpu() - x6.grad).abs().max()) < 1e-5 * max(1.0, float(g6.abs().max()))
    assert rel_err(g.grad, g6.grad) < 1e-5
    # keys broadcast over the batch: their gradient is the sum over it
    q, k, v = rn(3, 3, 10, 2, 16), rn(4, 1, 12, 2, 16), rn(5, 1, 12, 2, 16)
    qd, kd, vd = (t.to(DEV).requires_grad_(True) for t in (q, k, v))
    tokens.attention(qd, kd.expand(3, -1, -1, -1), vd.expand(3, -1, -1, -1)).sum().backward()
    q6, k6, v6 = (t.double().requires_grad_(True) for t in (q, k, v))
    s = torch.einsum("bihd,xjhd->bhij", q6, k6) / 4.0
    torch.einsum("bhij,xjhd->bihd", torch.softmax(s, -1), v6).sum().backward()
    for a, b in ((qd, q6), (kd, k6), (vd, v6)):
        assert a.grad.shape == b.grad.shape and float((a.grad.double().cpu() - b.grad).abs().max()) < 1e-5 * max(1.0, float(b.grad.abs().max()))
    # one tensor as query, key and value
    z = rn(6, 2, 8, 2, 16)
    zd, z6 = z.to(DEV).requires_grad_(True), z.double().requires_grad_(True)
    tokens.attention(zd, zd, zd, causal=True).square().sum().backward()
    s = (torch.einsum("bihd,bjhd->bhij", z6, z6) / 4.0).masked_fill(torch.ones(8, 8, dtype=torch.bool).triu(1), -math.inf)
    torch.einsum("bhij,bjhd->bihd", torch.softmax(s, -1), z6).square().sum().backward()
    assert rel_err(zd.grad, z6.grad) < 1e-5
    # without gradients nothing is saved
    with torch.no_grad():
        assert not tokens.attention(qd, kd.expand(3, -1, -1, -1), vd.expand(3, -1, -1, -1)).requires_grad


def test_attention_over_sliding_windows_of_one_tensor():
    """Keys whose rows share memory (overlapping windows): read in place without gradients, copied for them; the gradient sums what the windows share."""
    from pdae_amd import tokens
    q, base = rn(1, 3, 6, 2, 16), rn(2, 10, 2, 16)
    windows = lambda t: t.as_strided((3, 6, 2, 16), (64, 32, 16, 1))                                  # two tokens further each: windows share four of six
    qd, bd = q.to(DEV).requires_grad_(True), base.to(DEV).requires_grad_(True)
    o = tokens.attention(qd, windows(bd), windows(bd))
    with torch.no_grad():
        assert torch.equal(o, tokens.attention(qd, windows(bd), windows(bd)))
    o.square().sum().backward()
    q6, b6 = q.double().requires_grad_(True), base.double().requires_grad_(True)
    w6 = torch.stack([b6[2 * i:2 * i + 6] for i in range(3)])
    s = torch.einsum("bihd,bjhd->bhij", q6, w6) / 4.0
    torch.einsum("bhij,bjhd->bihd", torch.softmax(s, -1), w6).square().sum().backward()
    assert rel_err(qd.grad, q6.grad) < 1e-5 and rel_err(bd.grad, b6.grad) < 1e-5


@pytest.mark.parametrize("name", ["layer_norm", "dropout", "attention"])
def test_gradients_of_gradients_are_refused(name):
    """The backward is one kernel that autograd does not see into: a second derivative would silently miss terms."""
    from pdae_amd import tokens
    x = rn(3, 1, 5, 2, 16).to(DEV).requires_grad_(True)
    y = {"layer_norm": lambda: tokens.layer_norm(x), "dropout": lambda: tokens.dropout(x, 0.3, 1), "attention": lambda: tokens.attention(x, x, x)}[name]()
    g, = torch.autograd.grad(y.square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.square().sum().backward()


def test_functions_refuse_what_they_cannot_do():
    from pdae_amd import tokens
    from pdae_amd.hip import PdaeError
    x = torch.zeros(2, 4, 2, 8, device=DEV)
    for call in (lambda: tokens.layer_norm(x.half()), lambda: tokens.layer_norm(x, torch.ones(9, device=DEV)), lambda: tokens.layer_norm(x, torch.ones(8, device=DEV).bfloat16()),
                 lambda: tokens.dropout(x, 1.0, 0), lambda: tokens.dropout(x, 0.1, 0, residual=x.bfloat16()), lambda: tokens.attention(x, x, x.bfloat16()),
                 lambda: tokens.attention(x, x[:, :, :, :4], x[:, :, :, :4]), lambda: tokens.attention(x, x, x, k_len=torch.zeros(2, device=DEV)),
                 lambda: tokens.attention(x, x, x, k_len=torch.zeros(2, dtype=torch.int32)), lambda: tokens.attention(x, x, x, scale=-1.0),
                 lambda: tokens.attention(torch.zeros(1, 2, 1, 130, device=DEV), torch.zeros(1, 2, 1, 130, device=DEV), torch.zeros(1, 2, 1, 130, device=DEV))):
        with pytest.raises(PdaeError):
            call()


# ------------------------------------------------------------------------------------------------ streams and graphs
def _records(H, seed, train=True):
    """One pass of every operator over static buffers: (buffers that are written, op array, count)."""
    B, T, Hq, Hkv, D, Rr, Cc = 2, 150, 4, 2, 64, 70, 300
    r = lambda *s: rn(seed + len(s), *s).to(DEV)
    q, k, v, g = r(B, T, Hq, D), r(B, T, Hkv, D) * 1.1, r(B, T, Hkv, D) * 0.9, r(B, T, Hq, D) * 0.5
    q1, k1 = rn(seed, 1, 1, 8, D).to(DEV).bfloat16(), rn(seed + 1, 1, 2000, 1, D).to(DEV).bfloat16()
    a, a1 = H.Mha(B, T, T, Hq, Hkv, D, causal=True), H.Mha(1, 1, 2000, 8, 1, D, dtype=H.DT_BF16)
    x, dy, gm = r(Rr, Cc), r(Rr, Cc) * 0.7, r(Cc)
    out = dict(o=torch.empty_like(q), lse=torch.empty(B, Hq, T, device=DEV), dq=torch.empty_like(q), dk=torch.empty_like(k), dv=torch.empty_like(v), o1=torch.empty_like(q1),
               y=torch.empty_like(x), mean=torch.empty(Rr, device=DEV), rstd=torch.empty(Rr, device=DEV), dx=torch.empty_like(x), dg=torch.empty(Cc, device=DEV),
               db=torch.empty(Cc, device=DEV), z=torch.empty_like(x), dz=torch.empty_like(x))
    ws = [torch.empty(max(16, n), dtype=torch.uint8, device=DEV) for n in (a.ws_bytes(True), a1.ws_bytes(), H.layernorm_ws_bytes(Rr, Cc))]
    ops = [H.op_mha_fwd(a, q, k, v, out["o"], lse=out["lse"], ws=ws[0]), H.op_mha_bwd(a, q, k, v, out["o"], out["lse"], g, out["dq"], out["dk"], out["dv"], ws=ws[0]),
           H.op_mha_fwd(a1, q1, k1, k1, out["o1"], ws=ws[1]), H.op_layernorm_fwd(x, gm, None, Rr, Cc, 1e-5, out["y"], out["mean"], out["rstd"]),
           H.op_layernorm_bwd(x, gm, out["mean"], out["rstd"], dy, Rr, Cc, out["dx"], out["dg"], out["db"], ws[2]),
           H.op_dropout_fwd(out["y"], x, x.numel(), 0.1, out["z"], seed=seed, offset=3), H.op_dropout_bwd(dy, x.numel(), 0.1, out["dz"], seed=seed, offset=3)]
    return out, H.ops_array(ops), len(ops), (q, k, v, g, q1, k1, x, dy, gm, ws)


def test_captured_graph_replays_equal_the_eager_pass():
    """Forward and backward of all operators in one graph; other work and synchronisations between the replays, new inputs in place for the last one."""
    from pdae_amd import hip as H
    out, arr, n, keep = _records(H, 11)
    H.run_ops(arr, n)
    torch.cuda.synchronize()
    want = {k: v.clone() for k, v in out.items()}
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        H.run_ops(arr, n)
    for rep in range(4):
        for t in out.values():
            t.fill_(float("nan"))
        (torch.randn(512, 512, device=DEV) @ torch.randn(512, 512, device=DEV)).sum().item()
        graph.replay()
        torch.cuda.synchronize()
        for k in want:
            assert torch.equal(out[k], want[k]), (rep, k)
    keep[0].mul_(0.5)                                                     # new queries in the same buffer
    graph.replay()
    torch.cuda.synchronize()
    got = {k: v.clone() for k, v in out.items()}
    H.run_ops(arr, n)
    torch.cuda.synchronize()
    assert not torch.equal(got["o"], want["o"]) and all(torch.equal(got[k], out[k]) for k in got)


def test_two_streams_at_once_and_a_stream_that_is_not_current():
    from pdae_amd import hip as H
    sets = [_records(H, s) for s in (21, 33)]
    want = []
    for out, arr, n, _ in sets:
        H.run_ops(arr, n)
        torch.cuda.synchronize()
        want.append({k: v.clone() for k, v in out.items()})
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        for (out, arr, n, _k), st in zip(sets, streams):
            st.wait_stream(torch.cuda.current_stream())
            H.run_ops(arr, n, stream=st.cuda_stream)
        torch.cuda.synchronize()
        for (out, *_r), w in zip(sets, want):
            assert all(torch.equal(out[k], w[k]) for k in w)


def test_autograd_functions_run_on_the_current_stream():
    from pdae_amd import tokens
    q = rn(1, 2, 64, 2, 32).to(DEV).requires_grad_(True)
    tokens.attention(q, q, q).sum().backward()
    want = q.grad.clone()
    q.grad = None
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        tokens.attention(q, q, q).sum().backward()
    st.synchronize()
    assert torch.equal(q.grad, want)


# ------------------------------------------------------------------------------------------------ planned networks
def mlp_reference(sd, cfg, x, t, seed, step):
    """model/mlp_skip_net.py:67-78 with dropout behind the activation of every layer but the last, masks of stream (seed, step, layer i + 1)."""
    from oracle import pdae_oracle as O
    n, p = cfg["num_layers"], cfg["dropout"]
    cond = F.linear(O.timestep_embedding(t, cfg["time_emb_channel"]), sd["time_embed.0.weight"], sd["time_embed.0.bias"])
    cond = F.linear(F.silu(cond), sd["time_embed.2.weight"], sd["time_embed.2.bias"])
    h = x
    for i in range(n):
        h = F.linear(torch.cat([h, x], 1) if i else h, sd[f"layers.{i}.linear.weight"], sd[f"layers.{i}.linear.bias"])
        if i < n - 1:
            h = h * (1.0 + F.linear(F.silu(cond), sd[f"layers.{i}.linear_emb.weight"], sd[f"layers.{i}.linear_emb.bias"]))
            if cfg["use_norm"]:
                h = F.layer_norm(h, (h.shape[1],), sd[f"layers.{i}.norm.weight"], sd[f"layers.{i}.norm.bias"])
            h = F.silu(h)
            keep = R.keep_mask(h.numel(), p, seed, step, i + 1).view_as(h)
            h = torch.where(keep, h / (1 - p), torch.zeros_like(h))
    return h


@pytest.mark.parametrize("cfg,rows", [(dict(C.CFG_MLP, dropout=0.1), 6), (dict(input_channel=512, model_channel=2048, num_layers=4, time_emb_channel=64, use_norm=True, dropout=0.3), 16),
                                      (dict(input_channel=60, model_channel=90, num_layers=3, time_emb_channel=32, use_norm=False, dropout=0.5), 5)])
def test_mlp_skip_net_with_dropout_against_autograd(cfg, rows):
    """The tolerances of the same network without dropout (tests/test_networks_gpu.py): a kept element is multiplied once more."""
    from oracle import pdae_oracle as O
    from pdae_amd.model.mlp_skip_net import MLPSkipNet
    sd = O.synth_state_dict(O.mlp_skip_net_param_shapes(cfg), 7)
    net = MLPSkipNet(device=DEV, **cfg)
    net.load_state_dict(sd, strict=False)
    z, noise, t = rn(1, rows, cfg["input_channel"]), rn(2, rows, cfg["input_channel"]), torch.arange(rows) * 31
    random.seed(5)
    seed = random.getrandbits(31)
    ref_sd = {k: v.clone().requires_grad_(True) for k, v in sd.items()}
    zr = z.clone().requires_grad_(True)
    ref = mlp_reference(ref_sd, cfg, zr, t, seed, 0)
    (noise - ref).abs().mean().backward()
    net.train()
    zd = z.to(DEV).requires_grad_(True)
    random.seed(5)
    out = net(zd, t.to(DEV))
    assert rel_err(out, ref.detach()) < 1e-4
    (noise.to(DEV) - out).abs().mean().backward()
    G = net.grads()
    for k, v in ref_sd.items():
        assert rel_err(G[k], v.grad) < 2e-4, k
    assert rel_err(zd.grad, zr.grad) < 2e-4
    # evaluation, and training without gradients, drop nothing
    plain = O.mlp_skip_net_forward(sd, cfg, z, t)
    with torch.no_grad():
        assert rel_err(net(z.to(DEV), t.to(DEV)), plain) < 1e-4
    net.eval()
    assert rel_err(net(z.to(DEV), t.to(DEV)), plain) < 1e-4


def test_latent_training_step_with_dropout():
    """FusedLatentStep draws a new mask per step from the host's generator, and its gradients are those of the reference with that mask."""
    import copy
    from oracle import pdae_oracle as O
    from pdae_amd.diffusion.gaussian_diffusion import GaussianDiffusion
    from pdae_amd.model.mlp_skip_net import MLPSkipNet
    from pdae_amd.trainer.fused_step import FusedLatentStep
    cfg = dict(C.CFG_MLP, dropout=0.25)
    sd = O.synth_state_dict(O.mlp_skip_net_param_shapes(cfg), 3)
    gd = GaussianDiffusion({"timesteps": 1000, "betas_type": "linear"}, torch.device(DEV))
    z0, noise, t = rn(1, 8, 64), rn(2, 8, 64), torch.arange(8) * 90
    losses = []
    for run in range(2):
        net = MLPSkipNet(device=DEV, **cfg)
        net.load_state_dict(sd, strict=False)
        net.train()
        st = FusedLatentStep(gd, net, copy.deepcopy(net), 8, lr=0.0)
        random.seed(9)
        losses.append([float(st.step(z0.to(DEV), t=t.to(DEV), noise=noise.to(DEV))) for _ in range(3)])
    assert losses[0] == losses[1] and len(set(losses[0])) == 3            # repeatable, and a mask of its own per step (lr = 0: nothing else changes)
    random.seed(9)
    lc = gd.latent_diffusion_config
    sa, sb = lc["sqrt_alphas_cumprod"].cpu()[t][:, None], lc["sqrt_one_minus_alphas_cumprod"].cpu()[t][:, None]
    for step in range(3):
        ref = mlp_reference(sd, cfg, sa * z0 + sb * noise, t, random.getrandbits(31), step)
        want = float((noise - ref).abs().mean())
        assert abs(losses[0][step] - want) < 1e-4 * want


@pytest.mark.parametrize("N,S,Cc,heads,order", [(2, 12, 64, 1, False), (1, 32, 96, 2, True), (2, 4, 64, 4, False), (1, 20, 128, 4, False)])
def test_attention_block_at_any_size_equals_the_composed_path(monkeypatch, N, S, Cc, heads, order):
    """PDAE_ATTN_ANY=1: planned AttentionBlocks beyond the fused image kernels' shapes on pdae_mha_*, against GEMM + softmax (the default there): the bounds
    of the fused kernels' own comparison."""
    from pdae_amd import hip as H
    from pdae_amd.engine import Builder, Plan
    assert not H.attn_fused_ok(S * S, Cc, heads)
    P = {"a.norm.weight": rn(1, Cc, scale=0.1, shift=1.0), "a.norm.bias": rn(2, Cc, scale=0.1), "a.qkv.weight": rn(3, 3 * Cc, 1, 1, Cc, scale=1 / math.sqrt(Cc)),
         "a.qkv.bias": rn(4, 3 * Cc, scale=0.1), "a.proj_out.weight": rn(5, Cc, 1, 1, Cc, scale=1 / math.sqrt(Cc)), "a.proj_out.bias": rn(6, Cc, scale=0.1)}
    P = {k: v.to(DEV) for k, v in P.items()}
    x, dy = rn(7, N, S, S, Cc).to(DEV), rn(8, N, S, S, Cc).to(DEV)
    res = {}
    for flag in ("1", "0"):
        monkeypatch.setenv("PDAE_ATTN_ANY", flag)
        Gr = {k: torch.zeros_like(v) for k, v in P.items()}
        pl = Plan(DEV)
        B = Builder(pl, P, Gr, save=True)
        out, ctx = B.attention("a", x, heads, order)
        assert (ctx.mha is not None) == (flag == "1")
        dx, _ = B.attention_bwd(ctx, dy, need_dx=True)
        pl.compile().run()
        torch.cuda.synchronize()
        res[flag] = (out.clone(), dx.clone(), {k: v.clone() for k, v in Gr.items()})
    assert rel_err(res["1"][0], res["0"][0]) < 1e-5 and rel_err(res["1"][1], res["0"][1]) < 1e-5
    for k in P:
        assert rel_err(res["1"][2][k], res["0"][2][k]) < 2e-5, k
