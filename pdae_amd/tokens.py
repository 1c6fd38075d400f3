"""Tensor-level token operators with autograd: layer norm, dropout from a counter, attention over any number of tokens (include/pdae_hip.h:
pdae_layernorm_*, pdae_dropout_*, pdae_mha_*).

    h = tokens.layer_norm(x, gamma, beta)
    o = tokens.attention(q, k, v, causal=True)                 # [B, T, heads, D]
    x = tokens.dropout(h, p, seed, step, layer, residual=x)

Each function allocates its outputs, launches on the current stream of the tensors' device (which need not be the current device) and never
synchronises.  Activations are fp32 or bf16, parameters and their gradients fp32.  Host code that runs the same shapes every step builds op records
instead (hip.op_layernorm_fwd, ...) and keeps them in a Plan; that is also the form to capture into a graph (a backward through autograd can only be
captured together with its forward, and while no other graph of the same leaves lives).  Gradients of gradients are refused."""
import torch
from torch.autograd.function import once_differentiable

from . import hip as H


def _dtype(t, name):
    if t.dtype not in (torch.float32, torch.bfloat16):
        raise H.PdaeError(f"{name}: fp32 or bf16 expected, got {t.dtype}")
    return H.DTYPES[t.dtype]


def _on_device(name, first, *others):
    if first.device.type != "cuda":
        raise H.PdaeError(f"{name}: tensors must live on a ROCm device (no CPU fallback)")
    for t in others:
        if t is not None and t.device != first.device:
            raise H.PdaeError(f"{name}: tensors on {first.device} and {t.device}")
    return torch.cuda.device(first.device)


def _rows(x):
    """x as rows with contiguous channels: (tensor, rows, channels, row stride); a copy only when the strides do not allow rows."""
    if x.dim() == 0:
        raise H.PdaeError("layer_norm: a tensor of at least one dimension expected")
    C = x.shape[-1]
    if x.dim() == 2 and x.stride(1) == 1 and x.stride(0) >= C:
        return x, x.shape[0], C, x.stride(0)
    x = x.contiguous()
    return x, x.numel() // max(C, 1), C, C


def _fp32_vector(t, n, name):
    if t is not None and (t.dtype != torch.float32 or t.shape != (n,) or not t.is_contiguous()):
        raise H.PdaeError(f"{name}: contiguous fp32 [{n}] expected, got {t.dtype} {tuple(t.shape)}")


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        with _on_device("layer_norm", x, weight, bias):
            xr, R, C, ldx = _rows(x)
            _fp32_vector(weight, C, "layer_norm weight"); _fp32_vector(bias, C, "layer_norm bias")
            y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
            mean, rstd = (torch.empty(R, dtype=torch.float32, device=x.device) for _ in range(2))
            H.run(H.op_layernorm_fwd(xr, weight, bias, R, C, eps, y, mean, rstd, dtype=_dtype(x, "layer_norm"), ldx=ldx))
        ctx.save_for_backward(xr, weight, mean, rstd)
        ctx.has_bias, ctx.shape, ctx.ldx = bias is not None, x.shape, ldx
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        xr, weight, mean, rstd = ctx.saved_tensors
        with _on_device("layer_norm", xr, dy):
            dr, R, C, ldd = _rows(dy)
            dx = torch.empty(ctx.shape, dtype=xr.dtype, device=xr.device)
            dg = torch.empty(C, dtype=torch.float32, device=xr.device) if weight is not None and ctx.needs_input_grad[1] else None
            db = torch.empty(C, dtype=torch.float32, device=xr.device) if ctx.has_bias and ctx.needs_input_grad[2] else None
            ws = torch.empty(H.layernorm_ws_bytes(R, C), dtype=torch.uint8, device=xr.device) if dg is not None or db is not None else None
            H.run(H.op_layernorm_bwd(xr, weight, mean, rstd, dr, R, C, dx, dg, db, ws, dtype=_dtype(xr, "layer_norm"), ldx=ctx.ldx, lddy=ldd))
        return dx, dg, db, None


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """LayerNorm over the last dimension; weight / bias: fp32 [C] or None."""
    return _LayerNorm.apply(x, weight, bias, float(eps))


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, p, seed, step, layer):
        ctx.args = (p, seed, step, layer)
        with _on_device("dropout", x, residual):
            xc = x.contiguous()
            if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype):
                raise H.PdaeError("dropout: the residual must have x's shape and type")
            rc = None if residual is None else residual.contiguous()           # (a name of its own: the record holds its address only)
            y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
            H.run(H.op_dropout_fwd(xc, rc, x.numel(), p, y, seed=seed, offset=step, layer=layer, dtype=_dtype(x, "dropout")))
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        p, seed, step, layer = ctx.args
        with _on_device("dropout", dy):
            dc = dy.contiguous()
            dx = torch.empty(dy.shape, dtype=dy.dtype, device=dy.device)
            H.run(H.op_dropout_bwd(dc, dy.numel(), p, dx, seed=seed, offset=step, layer=layer, dtype=_dtype(dy, "dropout")))
        return dx, dy if ctx.needs_input_grad[1] else None, None, None, None, None


def dropout(x, p, seed, step=0, layer=0, residual=None):
    """(residual +) x with a fraction p of its elements dropped and the rest scaled by 1 / (1 - p).  The mask is a function of (seed, step, layer, element
    index): equal arguments give equal masks, and the backward regenerates it.  step and layer: 0 .. 2^32 - 1."""
    if not (0 <= int(step) < 1 << 32 and 0 <= int(layer) < 1 << 32):
        raise H.PdaeError(f"dropout: step {step} and layer {layer} must lie in [0, 2^32)")
    return _Dropout.apply(x, residual, float(p), int(seed), int(step), int(layer))


def _heads(t, group=1):
    """t ([B, T, H, D]) if the kernels take its strides, else a contiguous copy.  The limits are those of pdae_mha_desc: contiguous channels, token strides
    below 2^21 elements, and for queries whose `group` heads share a key head as rows of one tile (at most 128 of them) 2^28 over the group."""
    T, H = t.shape[1:3]
    if t.stride(3) != 1 or (T > 1 and t.stride(1) >= 1 << 21) or (group > 1 and H > 1 and T * group <= 128 and group * t.stride(2) >= 1 << 28):
        return t.contiguous()
    return t


def _own_rows(t):
    """No two rows of D channels of t share memory."""
    extent = t.shape[3]
    for s, n in sorted((s, n) for s, n in zip(t.stride()[:3], t.shape[:3]) if n > 1):
        if s < extent:
            return False
        extent += s * (n - 1)
    return True


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, q_len, k_len, causal, scale, need):
        with _on_device("attention", q, k, v, q_len, k_len):
            if q.dim() != 4 or k.dim() != 4 or k.shape != v.shape or q.shape[0] != k.shape[0] or q.shape[3] != k.shape[3]:
                raise H.PdaeError(f"attention: q [B, Tq, Hq, D] and k, v [B, Tk, Hkv, D] expected, got {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
            if k.dtype != q.dtype or v.dtype != q.dtype:
                raise H.PdaeError("attention: q, k and v must have one type")
            for t in (q_len, k_len):
                if t is not None and (t.dtype != torch.int32 or t.shape != (q.shape[0],) or not t.is_contiguous()):
                    raise H.PdaeError("attention: lengths must be contiguous int32 [B]")
            # gradients get their tensor's strides, so in training rows must not share memory (a tensor expanded over batch or heads, or of sliding windows, is
            # copied; autograd sums its copies' gradients)
            q, k, v = _heads(q, q.shape[2] // max(k.shape[2], 1)), _heads(k), _heads(v)
            if need:
                q, k, v = (t if _own_rows(t) else t.contiguous() for t in (q, k, v))
            B, Tq, Hq, D = q.shape
            o = torch.empty(B, Tq, Hq, D, dtype=q.dtype, device=q.device)
            a = H.Mha(B, Tq, k.shape[1], Hq, k.shape[2], D, dtype=_dtype(q, "attention"), causal=causal, scale=scale, q_stride=q.stride()[:3], k_stride=k.stride()[:3],
                      v_stride=v.stride()[:3], o_stride=o.stride()[:3])
            lse = torch.empty(B, Hq, Tq, dtype=torch.float32, device=q.device) if need else None
            n = a.ws_bytes(False)
            ws = torch.empty(n, dtype=torch.uint8, device=q.device) if n else None
            H.run(H.op_mha_fwd(a, q, k, v, o, lse=lse, q_len=q_len, k_len=k_len, ws=ws))
        if need:
            ctx.save_for_backward(q, k, v, o, lse, q_len, k_len)
            ctx.a = a
        return o

    @staticmethod
    @once_differentiable
    def backward(ctx, d_o):
        q, k, v, o, lse, q_len, k_len = ctx.saved_tensors
        a = ctx.a
        with _on_device("attention", q, d_o):
            d_o = d_o.contiguous()
            dq, dk, dv = (torch.empty_strided(t.shape, t.stride(), dtype=t.dtype, device=t.device) for t in (q, k, v))
            ws = torch.empty(max(16, a.ws_bytes(True)), dtype=torch.uint8, device=q.device)
            H.run(H.op_mha_bwd(a, q, k, v, o, lse, d_o, dq, dk, dv, q_len=q_len, k_len=k_len, ws=ws))
        return dq, dk, dv, None, None, None, None, None


def attention(q, k, v, q_len=None, k_len=None, causal=False, scale=None):
    """softmax(scale q k^T) v per head: q [B, Tq, Hq, D], k / v [B, Tk, Hkv, D] (Hq a multiple of Hkv, D <= 128), any token counts and strides with contiguous
    channels.  q_len / k_len: int32 [B] device tensors, rows behind them do not exist; causal: query i sees keys j <= i + k_len - q_len.  scale: 1 / sqrt(D)."""
    need = torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad)
    return _Attention.apply(q, k, v, q_len, k_len, bool(causal), scale, need)
