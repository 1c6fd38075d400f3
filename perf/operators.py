"""Token operators of pdae_amd, measured on their own: layer norm with its backward pass, dropout from a counter, attention over any number of
tokens with its backward pass and its single-token form.

`run` computes them in elementary torch operations in 32 bits (own = False) or with the framework's kernels (own = True); `exact` computes
them in 64 bits from the definitions.  Layouts are the framework's: token rows [rows][channels], heads [batch][token][head][channel]."""
import math

import numpy as np
import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "bf16": 2}


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one layer's normalisation in the latent denoiser's training step (128 latents, 2048 wide, 32-bit): launch latency counts
        dict(name="norm_latent", op="norm_train", dtype="f32", R=128, C=2048),
        # token rows of a training step in bf16, the memory-bound end
        dict(name="norm_tokens", op="norm_train", dtype="bf16", R=65536, C=1536),
        # sampling: forward only, a row length that no vector width divides
        dict(name="norm_odd", op="norm_fwd", dtype="bf16", R=9001, C=1027),
        # dropout behind the latent denoiser's activation
        dict(name="drop_latent", op="drop", dtype="f32", R=128, C=2048, p=0.1, res=False),
        # residual branch of a token block in training, odd sizes
        dict(name="drop_residual", op="drop", dtype="bf16", R=40007, C=1027, p=0.1, res=True),
        # one small attention call: the 8 x 8 level of a small network, latency
        dict(name="attn_small", op="attn_fwd", dtype="f32", B=2, Hq=1, Hkv=1, Tq=64, Tk=64, D=32, causal=False, ragged=False),
        # the 32 x 32 level in the framework's own type, four heads of 64, training
        dict(name="attn_f32_train", op="attn_train", dtype="f32", B=8, Hq=4, Hkv=4, Tq=1024, Tk=1024, D=64, causal=False, ragged=False),
        # sampling at 64 x 64 tokens in bf16
        dict(name="attn_sample", op="attn_fwd", dtype="bf16", B=4, Hq=8, Hkv=8, Tq=4096, Tk=4096, D=64, causal=False, ragged=False),
        # the largest: causal training over long rows, heads of 128
        dict(name="attn_long_train", op="attn_train", dtype="bf16", B=4, Hq=16, Hkv=16, Tq=4096, Tk=4096, D=128, causal=True, ragged=False),
        # a padded batch with shared key / value heads, odd head width and lengths, one empty sample
        dict(name="attn_ragged_train", op="attn_train", dtype="bf16", B=7, Hq=12, Hkv=3, Tq=1501, Tk=1733, D=72, causal=True, ragged=True),
        # cross-attention of many pixels onto a short condition
        dict(name="attn_cross", op="attn_fwd", dtype="bf16", B=16, Hq=8, Hkv=8, Tq=1024, Tk=77, D=40, causal=False, ragged=False),
        # one new token per sample against a long, ragged cache with shared heads
        dict(name="attn_token", op="attn_fwd", dtype="bf16", B=24, Hq=32, Hkv=8, Tq=1, Tk=8191, D=128, causal=True, ragged=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    dtype = rng.choice(["f32", "bf16"])
    kind = rng.choice(["norm_train", "norm_fwd", "drop", "attn_fwd", "attn_train", "attn_train", "attn_token"])
    if kind.startswith("norm") or kind == "drop":
        C = _log(rng, 64, 4096)
        R = _log(rng, 16, (65536 * 1536 // 2) // C if dtype == "f32" else 65536 * 1536 // C)
        case = dict(op=kind, dtype=dtype, R=R, C=C)
        if kind == "drop":
            case["R"] = min(case["R"], 40007 * 1027 // C)
            case.update(p=rng.choice([0.05, 0.1, 0.25, 0.5]), res=rng.random() < 0.5)
        return case
    D = rng.choice([32, 40, 64, 72, 80, 96, 128])
    Hkv = rng.choice([1, 2, 3, 4, 8])
    Hq = Hkv * rng.choice([1, 1, 2, 4])
    causal, ragged = rng.random() < 0.5, rng.random() < 0.5
    if kind == "attn_token":
        return dict(op="attn_fwd", dtype=dtype, B=_log(rng, 1, 24), Hq=Hq, Hkv=Hkv, Tq=rng.choice([1, 1, 2, 4]), Tk=_log(rng, 64, 8191), D=D, causal=causal,
                    ragged=ragged)
    Tq = _log(rng, 16, 4096)
    Tk = Tq if rng.random() < 0.6 else _log(rng, 16, 4096)
    most = 2.0e9 if dtype == "bf16" else 3.0e7                     # scores of the largest listed cases
    B = max(1, min(_log(rng, 1, 16), int(most // (2 * Hq * Tq * Tk))))
    Hq, Hkv = (Hq, Hkv) if B * Hq * Tq * Tk <= most else (1, 1)
    return dict(op=kind, dtype=dtype, B=B, Hq=Hq, Hkv=Hkv, Tq=Tq, Tk=Tk, D=D, causal=causal, ragged=ragged)


def _lengths(case):
    """(query lengths, key lengths) of the batch: a padded batch has a full, an empty and in-between samples (one token per sample keeps its token)."""
    B, Tq, Tk = case["B"], case["Tq"], case["Tk"]
    if not case["ragged"]:
        return [Tq] * B, [Tk] * B
    part = [1.0 if b == 0 else 0.0 if b == B - 1 else (0.61803399 * b) % 1.0 for b in range(B)]
    return ([Tq] * B if Tq <= 4 else [int(round(f * Tq)) for f in part]), [int(round(f * Tk)) for f in part]


def _pairs(case):
    """(query, key) pairs of all samples, one head, that the masks leave."""
    n = 0
    for lq, lk in zip(*_lengths(case)):
        if case["causal"]:
            first = lk - lq + 1                                     # keys that query 0 sees (may be negative)
            lo, hi = max(first, 0), first + lq - 1                  # ... and the last query
            n += (lo + hi) * (hi - lo + 1) // 2 if lq and hi >= lo else 0
        else:
            n += lq * lk
    return n


def work(case):
    s = SIZE[case["dtype"]]
    if case["op"] in ("norm_fwd", "norm_train"):
        n = case["R"] * case["C"]
        if case["op"] == "norm_fwd":
            return {"bytes": 2 * n * s + 8 * case["C"] + 8 * case["R"], "flops": 8 * n}
        return {"bytes": 4 * n * s + 20 * case["C"] + 8 * case["R"], "flops": 20 * n}      # x, dy in; y, dx out; gamma, beta and their gradients
    if case["op"] == "drop":
        n = case["R"] * case["C"]
        return {"bytes": (5 if case["res"] else 4) * n * s, "flops": 4 * n}
    D, Hq, Hkv = case["D"], case["Hq"], case["Hkv"]
    lq, lk = (sum(v) for v in _lengths(case))
    pairs, B = _pairs(case) * Hq, case["B"]
    q, kv, o = lq * Hq * D, lk * Hkv * D, B * case["Tq"] * Hq * D                            # padded rows are read by nobody, and written
    if case["op"] == "attn_fwd":
        return {"bytes": (q + 2 * kv + o) * s, "flops": 4 * pairs * D}
    dkv = B * case["Tk"] * Hkv * D
    return {"bytes": (2 * q + 2 * kv + 2 * o + 2 * dkv) * s + 4 * B * Hq * case["Tq"], "flops": 14 * pairs * D}


# ------------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed) * 2654435761 % (1 << 62) + 17)
    dt = TYPES[case["dtype"]]

    def rn(*shape, scale=1.0, shift=0.0):
        return (torch.randn(*shape, generator=g, device=DEV) * scale + shift).to(dt)

    st = dict(case=dict(case), seed=int(seed))
    if case["op"] in ("norm_fwd", "norm_train"):
        R, C = case["R"], case["C"]
        st.update(x=rn(R, C, scale=1.5, shift=0.3), dy=rn(R, C), gamma=torch.randn(C, generator=g, device=DEV) * 0.1 + 1.0,
                  beta=torch.randn(C, generator=g, device=DEV) * 0.1)
        return st
    if case["op"] == "drop":
        R, C = case["R"], case["C"]
        st.update(x=rn(R, C), dy=rn(R, C), res=rn(R, C) if case["res"] else None, drop_seed=1000003 * int(seed) + 11, drop_step=int(seed) % 9973)
        return st
    B, Hq, Hkv, Tq, Tk, D = (case[n] for n in ("B", "Hq", "Hkv", "Tq", "Tk", "D"))
    st.update(q=rn(B, Tq, Hq, D, scale=1.3), k=rn(B, Tk, Hkv, D, scale=1.3), v=rn(B, Tk, Hkv, D), d_o=rn(B, Tq, Hq, D) if case["op"] == "attn_train" else None)
    lq, lk = _lengths(case)
    st.update(q_len=torch.tensor(lq, dtype=torch.int32, device=DEV), k_len=torch.tensor(lk, dtype=torch.int32, device=DEV))
    return st


# ------------------------------------------------------------------------------------------------ the plain form
def _plain_norm(st):
    c = st["case"]
    dt = TYPES[c["dtype"]]
    x, gamma, beta = st["x"].float(), st["gamma"], st["beta"]
    mean = x.mean(dim=1, keepdim=True)
    d = x - mean
    rstd = 1.0 / torch.sqrt((d * d).mean(dim=1, keepdim=True) + 1e-5)
    xh = d * rstd
    y = (xh * gamma + beta).to(dt)
    out = dict(y=y, mean=mean[:, 0], rstd=rstd[:, 0])
    if c["op"] == "norm_train":
        dy = st["dy"].float()
        g = dy * gamma
        dx = rstd * (g - g.mean(dim=1, keepdim=True) - xh * (g * xh).mean(dim=1, keepdim=True))
        out.update(dx=dx.to(dt), dgamma=(dy * xh).sum(dim=0), dbeta=dy.sum(dim=0))
    return out


def _plain_keep(n, p, seed, step):
    """Keep mask of n elements: Philox2x32, ten rounds; one counter per four elements, 16 bits each."""
    m32 = 0xFFFFFFFF
    quad = torch.arange((n + 3) // 4, device=DEV, dtype=torch.int64)
    a = quad & m32
    b = (step & m32) ^ (((quad >> 32) * 0x85EBCA6B) & m32)
    key = (seed & m32) ^ (((seed >> 32) * 0xC2B2AE35) & m32) ^ (((step >> 32) * 0x27D4EB2F) & m32)
    for _ in range(10):
        prod = a * 0xD256D193                                       # wraps modulo 2^64: the low and the high word come out right
        a, b = ((prod >> 32) & m32) ^ key ^ b, prod & m32
        key = (key + 0x9E3779B9) & m32
    u = torch.stack([a & 0xFFFF, a >> 16, b & 0xFFFF, b >> 16], dim=1).reshape(-1)[:n]
    return u >= int(p * 65536.0 + 0.5)


def _plain_drop(st):
    c = st["case"]
    dt = TYPES[c["dtype"]]
    keep = _plain_keep(st["x"].numel(), c["p"], st["drop_seed"], st["drop_step"]).view_as(st["x"])
    f = keep.float() * (1.0 / (1.0 - c["p"]))
    y = st["x"].float() * f
    if st["res"] is not None:
        y = y + st["res"].float()
    return dict(y=y.to(dt), dx=(st["dy"].float() * f).to(dt))


def _plain_attn(st):
    c = st["case"]
    dt = TYPES[c["dtype"]]
    B, Hq, Hkv, Tq, Tk, D = (c[n] for n in ("B", "Hq", "Hkv", "Tq", "Tk", "D"))
    G, scale = Hq // Hkv, 1.0 / math.sqrt(D)

    def heads(t, T, H):                                             # -> [B * Hkv, (G *) T, D]
        t = t.float().permute(0, 2, 1, 3)
        return t.reshape(B * Hkv, (H // Hkv) * T, D)

    q, k, v = heads(st["q"], Tq, Hq), heads(st["k"], Tk, Hkv), heads(st["v"], Tk, Hkv)
    i, j = torch.arange(Tq, device=DEV), torch.arange(Tk, device=DEV)
    lq, lk = st["q_len"].long()[:, None, None], st["k_len"].long()[:, None, None]
    ok = (i[None, :, None] < lq) & (j[None, None, :] < lk)          # [B, Tq, Tk]
    if c["causal"]:
        ok = ok & (j[None, None, :] <= i[None, :, None] + lk - lq)
    ok = ok[:, None, None].expand(B, Hkv, G, Tq, Tk).reshape(B * Hkv, G * Tq, Tk)
    s = torch.matmul(q, k.transpose(1, 2).contiguous()) * scale
    s = s.masked_fill(~ok, -math.inf)
    m = s.amax(dim=2, keepdim=True)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    p = torch.exp(s - m)
    del s
    total = p.sum(dim=2, keepdim=True)
    lse = torch.where(total > 0, m + torch.log(total), torch.full_like(m, -math.inf))
    p = p / torch.where(total > 0, total, torch.ones_like(total))
    o = torch.matmul(p, v)

    def back(t, T, H):
        return t.view(B, H, T, D).permute(0, 2, 1, 3).contiguous().to(dt)

    if c["op"] == "attn_fwd":
        return dict(o=back(o, Tq, Hq))
    d_o = heads(st["d_o"], Tq, Hq)
    dv = torch.matmul(p.transpose(1, 2).contiguous(), d_o)
    dp = torch.matmul(d_o, v.transpose(1, 2).contiguous())
    ds = p * (dp - (p * dp).sum(dim=2, keepdim=True)) * scale
    del p, dp
    return dict(o=back(o, Tq, Hq), lse=lse.view(B, Hq, Tq), dq=back(torch.matmul(ds, k), Tq, Hq),
                dk=back(torch.matmul(ds.transpose(1, 2).contiguous(), q), Tk, Hkv), dv=back(dv, Tk, Hkv))


# ------------------------------------------------------------------------------------------------ the framework's kernels
def _plan(st):
    """The op records of one pass over the state's buffers: what a planned network keeps (pdae_amd.engine.Plan holds the same array)."""
    from pdae_amd import hip as H
    c = st["case"]
    dt = TYPES[c["dtype"]]
    kind = H.DTYPES[c["dtype"]]
    if c["op"] in ("norm_fwd", "norm_train"):
        R, C = c["R"], c["C"]
        out = dict(y=torch.empty(R, C, dtype=dt, device=DEV), mean=torch.empty(R, device=DEV), rstd=torch.empty(R, device=DEV))
        ops = [H.op_layernorm_fwd(st["x"], st["gamma"], st["beta"], R, C, 1e-5, out["y"], out["mean"], out["rstd"], dtype=kind)]
        if c["op"] == "norm_train":
            out.update(dx=torch.empty(R, C, dtype=dt, device=DEV), dgamma=torch.empty(C, device=DEV), dbeta=torch.empty(C, device=DEV))
            st["ws"] = torch.empty(H.layernorm_ws_bytes(R, C), dtype=torch.uint8, device=DEV)
            ops.append(H.op_layernorm_bwd(st["x"], st["gamma"], out["mean"], out["rstd"], st["dy"], R, C, out["dx"], out["dgamma"], out["dbeta"], st["ws"],
                                          dtype=kind))
    elif c["op"] == "drop":
        n = st["x"].numel()
        out = dict(y=torch.empty_like(st["x"]), dx=torch.empty_like(st["x"]))
        ops = [H.op_dropout_fwd(st["x"], st["res"], n, c["p"], out["y"], seed=st["drop_seed"], offset=st["drop_step"], dtype=kind),
               H.op_dropout_bwd(st["dy"], n, c["p"], out["dx"], seed=st["drop_seed"], offset=st["drop_step"], dtype=kind)]
    else:
        B, Hq, Hkv, Tq, Tk, D = (c[n] for n in ("B", "Hq", "Hkv", "Tq", "Tk", "D"))
        a = H.Mha(B, Tq, Tk, Hq, Hkv, D, dtype=kind, causal=c["causal"])
        train = c["op"] == "attn_train"
        lens = (st["q_len"], st["k_len"]) if c["ragged"] else (None, None)
        out = dict(o=torch.empty_like(st["q"]))
        if train:
            out.update(lse=torch.empty(B, Hq, Tq, device=DEV), dq=torch.empty_like(st["q"]), dk=torch.empty_like(st["k"]), dv=torch.empty_like(st["v"]))
        st["ws"] = torch.empty(max(16, a.ws_bytes(train)), dtype=torch.uint8, device=DEV)
        ops = [H.op_mha_fwd(a, st["q"], st["k"], st["v"], out["o"], lse=out.get("lse"), q_len=lens[0], k_len=lens[1], ws=st["ws"])]
        if train:
            ops.append(H.op_mha_bwd(a, st["q"], st["k"], st["v"], out["o"], out["lse"], st["d_o"], out["dq"], out["dk"], out["dv"], q_len=lens[0], k_len=lens[1],
                                    ws=st["ws"]))
    st["out"], st["n_ops"], st["ops"], st["run_ops"] = out, len(ops), H.ops_array(ops), H.run_ops


def run(state):
    if own:
        if "ops" not in state:
            _plan(state)
        state["run_ops"](state["ops"], state["n_ops"])
        return state["out"]
    op = state["case"]["op"]
    return _plain_drop(state) if op == "drop" else _plain_norm(state) if op.startswith("norm") else _plain_attn(state)


# ------------------------------------------------------------------------------------------------ the definitions in 64 bits
def _exact_keep(n, p, seed, step):
    mask = np.uint64(0xFFFFFFFF)
    q = np.arange((n + 3) // 4, dtype=np.uint64)
    c0, c1 = q & mask, np.uint64(step & 0xFFFFFFFF) ^ (((q >> np.uint64(32)) * np.uint64(0x85EBCA6B)) & mask)
    key = (seed ^ ((seed >> 32) * 0xC2B2AE35) ^ ((step >> 32) * 0x27D4EB2F)) & 0xFFFFFFFF
    for _ in range(10):
        prod = c0 * np.uint64(0xD256D193)
        c0, c1 = (prod >> np.uint64(32)) ^ np.uint64(key) ^ c1, prod & mask
        key = (key + 0x9E3779B9) & 0xFFFFFFFF
    words = np.empty((len(q), 2), dtype="<u4")
    words[:, 0], words[:, 1] = c0, c1
    return words.view("<u2").reshape(-1)[:n] >= int(p * 65536.0 + 0.5)


def exact(case, seed):
    st = prepare(case, seed)
    f64 = torch.float64
    if case["op"] == "drop":
        keep = torch.from_numpy(_exact_keep(st["x"].numel(), case["p"], st["drop_seed"], st["drop_step"])).to(DEV).view_as(st["x"])
        y = torch.where(keep, st["x"].to(f64) / (1.0 - case["p"]), 0.0)
        return dict(y=y if st["res"] is None else y + st["res"].to(f64), dx=torch.where(keep, st["dy"].to(f64) / (1.0 - case["p"]), 0.0))
    if case["op"].startswith("norm"):
        x, dy, C = st["x"].to(f64), st["dy"].to(f64), case["C"]
        mean = x.sum(1) / C
        var = ((x - mean[:, None]) ** 2).sum(1) / C
        rstd = (var + 1e-5) ** -0.5
        xh = (x - mean[:, None]) * rstd[:, None]
        out = dict(y=xh * st["gamma"].to(f64) + st["beta"].to(f64), mean=mean, rstd=rstd)
        if case["op"] == "norm_train":
            g = dy * st["gamma"].to(f64)
            s1, s2 = g.sum(1), (g * xh).sum(1)
            out.update(dx=(C * g - s1[:, None] - xh * s2[:, None]) * (rstd / C)[:, None], dgamma=(dy * xh).sum(0), dbeta=dy.sum(0))
        return out
    B, Hq, Hkv, Tq, Tk, D = (case[n] for n in ("B", "Hq", "Hkv", "Tq", "Tk", "D"))
    train = case["op"] == "attn_train"
    lq, lk = _lengths(case)
    o = torch.zeros(B, Tq, Hq, D, dtype=f64, device=DEV)
    if train:
        lse = torch.full((B, Hq, Tq), -math.inf, dtype=f64, device=DEV)
        dq, dk, dv = torch.zeros_like(o), torch.zeros(B, Tk, Hkv, D, dtype=f64, device=DEV), torch.zeros(B, Tk, Hkv, D, dtype=f64, device=DEV)
    for b in range(B):
        n, m = lq[b], lk[b]
        if not n or not m:
            continue
        hidden = None
        if case["causal"]:
            hidden = torch.ones(n, m, dtype=torch.bool, device=DEV).triu(m - n + 1)
        for h in range(Hq):
            kv = h // (Hq // Hkv)
            q, k, v = (t.to(f64) for t in (st["q"][b, :n, h], st["k"][b, :m, kv], st["v"][b, :m, kv]))
            s = torch.mm(q, k.t().contiguous()) / D ** 0.5
            if hidden is not None:
                s.masked_fill_(hidden, -math.inf)
            z = torch.logsumexp(s, dim=1)
            p = torch.exp(s - z[:, None]).masked_fill_((z == -math.inf)[:, None], 0.0)
            o[b, :n, h] = torch.mm(p, v)
            if train:
                lse[b, h, :n] = z
                go = st["d_o"][b, :n, h].to(f64)
                dv[b, :m, kv] += torch.mm(p.t().contiguous(), go)
                ds = p * (torch.mm(go, v.t().contiguous()) - (go * o[b, :n, h]).sum(1, keepdim=True)) / D ** 0.5
                dq[b, :n, h] = torch.mm(ds, k)
                dk[b, :m, kv] += torch.mm(ds.t().contiguous(), q)
    return dict(o=o, lse=lse, dq=dq, dk=dk, dv=dv) if train else dict(o=o)
