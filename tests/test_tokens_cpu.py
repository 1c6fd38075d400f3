"""CPU: what the tensor functions of pdae_amd/tokens.py hand to the kernels -- buffers, their types and how long they live, and which layouts are copied.  Nothing is
launched: the op records are caught where they would run."""
import contextlib

import pytest
import torch


@pytest.fixture
def caught(monkeypatch):
    """Lets the functions run on CPU tensors: [(op constructor, args, kwargs)] of every record built, `ran` called in place of the launch."""
    from pdae_amd import tokens

    class Caught(list):
        def ran(self, op):
            pass
    calls = Caught()
    monkeypatch.setattr(tokens, "_on_device", lambda name, first, *others: contextlib.nullcontext())

    class Hip:
        def __getattr__(self, name):
            f = getattr(tokens_hip, name)
            if not name.startswith("op_"):
                return f

            def build(*a, **k):
                calls.append((name, a, k))
                return f(*a, **k)
            return build

        def run(self, op, stream=None):
            calls.ran(op)
    tokens_hip = tokens.H
    monkeypatch.setattr(tokens, "H", Hip())
    return calls


@pytest.mark.parametrize("default", [torch.bfloat16, torch.float16, torch.float64])
def test_statistics_and_parameter_gradients_are_fp32_under_any_default_type(caught, default):
    """The kernels write fp32 statistics and parameter gradients: a buffer of torch's default type would be written past its end (bf16) or read as garbage."""
    from pdae_amd import tokens
    x = torch.zeros(3, 8, dtype=torch.bfloat16, requires_grad=True)
    w, b = (torch.ones(8, dtype=torch.float32, requires_grad=True) for _ in range(2))
    q = torch.zeros(1, 4, 2, 8, dtype=torch.bfloat16, requires_grad=True)
    before = torch.get_default_dtype()
    torch.set_default_dtype(default)
    try:
        y = tokens.layer_norm(x, w, b)
        y.backward(torch.zeros_like(y))
        o = tokens.attention(q, q, q)
        o.backward(torch.zeros_like(o))
    finally:
        torch.set_default_dtype(before)
    args = {n: (a, k) for n, a, k in caught}
    fp32 = list(args["op_layernorm_fwd"][0][7:9]) + list(args["op_layernorm_bwd"][0][8:10]) + [args["op_mha_fwd"][1]["lse"]]
    assert len(fp32) == 5 and all(t.dtype == torch.float32 for t in fp32)
    assert y.dtype == o.dtype == torch.bfloat16 and w.grad.dtype == torch.float32


def test_no_buffer_of_the_package_takes_torchs_default_type():
    """Every kernel argument has a fixed element type: a factory call that names none follows torch.set_default_dtype, and the kernel writes past the buffer."""
    import ast
    import os
    import pdae_amd
    root, bad = os.path.dirname(pdae_amd.__file__), []
    for folder, _, files in os.walk(root):
        for f in files:
            if not f.endswith(".py"):
                continue
            path = os.path.join(folder, f)
            with open(path) as fh:
                tree = ast.parse(fh.read())
            for n in ast.walk(tree):
                if isinstance(n, ast.Call) and isinstance(n.func, ast.Attribute) and isinstance(n.func.value, ast.Name) and n.func.value.id == "torch" and \
                        n.func.attr in ("empty", "zeros", "ones", "full", "rand", "randn", "empty_strided") and "dtype" not in [k.arg for k in n.keywords]:
                    bad.append(f"{os.path.relpath(path, root)}:{n.lineno}")
    assert not bad, bad


def test_contiguous_copies_live_until_the_launch(caught):
    """A record holds addresses: a copy that is dropped before the record runs may be handed to another thread of the same stream, which then writes into it."""
    import weakref

    from pdae_amd import tokens
    base = torch.randn(8, 6)
    refs = []

    def ran(op):
        while caught:                                     # (the fixture's own hold on the arguments ends here)
            refs.extend(weakref.ref(t) for t in caught.pop()[1] if isinstance(t, torch.Tensor))
        assert refs and all(r() is not None for r in refs)
    caught.ran = ran
    tokens.dropout(base.t(), 0.1, 1, residual=(base * 2).t())
    assert len(refs) == 3


def test_layouts_the_kernels_take_are_not_copied():
    """A head-major cache has head strides of tokens x channels: only token strides (and packed query heads) are limited in the kernels."""
    from pdae_amd import tokens
    meta = lambda *s: torch.empty(*s, dtype=torch.bfloat16, device="meta")
    cache = meta(2, 8, 8192, 128).transpose(1, 2)
    assert cache.stride() == (8 << 20, 128, 1 << 20, 1) and tokens._heads(cache) is cache
    q = meta(2, 32, 1, 128).transpose(1, 2)
    assert tokens._heads(q, group=4) is q
    one = meta(1, 512, 32, 128).transpose(0, 1)                                        # the stride of a lone token is no limit
    assert tokens._heads(one, group=4) is one
    wide = meta(2, 4, 1 << 21)[:, :, :16].unflatten(2, (2, 8))                         # token stride 2^21: beyond the kernels' tile
    assert tokens._heads(wide).is_contiguous()
    apart = torch.empty_strided((1, 4, 2, 8), (0, 8, 1 << 27, 1), device="meta")       # two packed query heads 2^27 apart
    assert tokens._heads(apart) is apart and tokens._heads(apart, group=2).is_contiguous()
    many = torch.empty_strided((1, 65, 2, 8), (0, 8, 1 << 27, 1), device="meta")       # 65 x 2 rows: heads are not packed
    assert tokens._heads(many, group=2) is many
    assert tokens._heads(meta(2, 4, 8, 2).transpose(2, 3)).is_contiguous()             # channels apart


def test_layer_norm_of_a_scalar_is_refused(caught):
    from pdae_amd import tokens
    from pdae_amd.hip import PdaeError
    with pytest.raises(PdaeError, match="dimension"):
        tokens.layer_norm(torch.zeros(()))
