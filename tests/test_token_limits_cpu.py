"""CPU: what the C entries of the token operators refuse, and what they must not refuse."""
import pytest


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


def test_strides_of_one_element_axes_are_not_looked_at(H):
    """A tensor with one sample, token or head may carry any stride there (time-major queries of one token, a slice of a cache): the address never uses it."""
    far = 1 << 45
    one = H.Mha(1, 1, 1, 1, 1, 128, **{k + "_stride": (far, far, far) for k in "qkvo"})
    refuses(H, H.op_mha_fwd(one, None, P, P, P), "null")
    refuses(H, H.op_mha_bwd(one, P, P, P, P, P, P, None, P, P, ws=P, ws_bytes=1 << 40), "null")
    # one token of 512 samples, samples inside the token: contiguous, with a token stride of 512 x 32 x 128
    t = H.Mha(512, 1, 64, 32, 32, 128, dtype=H.DT_BF16, q_stride=(4096, 1 << 21, 128))
    refuses(H, H.op_mha_fwd(t, None, P, P, P), "null")
    # a shared key head with one query head has no packed rows
    g = H.Mha(2, 4, 4, 1, 1, 8, q_stride=(64, 16, 1 << 30))
    refuses(H, H.op_mha_fwd(g, None, P, P, P), "null")
    # where the axis is longer the limits stand
    for k, s in (("q", (4096, 1 << 21, 128)), ("k", (4096, 1 << 21, 128))):
        refuses(H, H.op_mha_fwd(H.Mha(1, 2, 2, 2, 2, 8, **{k + "_stride": s}), P, P, P, P), "token stride")
    refuses(H, H.op_mha_fwd(H.Mha(2, 1, 1, 1, 1, 8, v_stride=(far, 1, 1)), P, P, P, P), "out of range")
    refuses(H, H.op_mha_fwd(H.Mha(1, 1, 4, 2, 1, 8, q_stride=(1, 1, 1 << 27)), P, P, P, P), "head stride")


def test_attention_is_refused_before_anything_is_launched(H):
    """Every size check stands in front of the first launch: a refused backward has not written dq or the workspace.  (Here a launch ends in another error.)"""
    a = H.Mha(1, 1, (1 << 30) - 1, 2, 2, 8)                                # 2^23 key tiles of two heads
    bwd = H.op_mha_bwd(a, P, P, P, P, P, P, P, P, P, ws=P, ws_bytes=1 << 60)
    refuses(H, bwd, "too many")


def test_gradients_in_the_place_of_what_is_still_read_are_refused(H):
    """Layer norm up to 1024 rows: blocks of columns read x and dy beside the blocks that write dx, and attention's second kernel reads what the first has written
    over -- in place they gave wrong weight gradients without a word."""
    W, Q = 1 << 20, P + 4096
    refuses(H, H.op_layernorm_fwd(P, P, P, 4, 8, 1e-5, P, ldx=8, ldy=9), "in the place of")      # (with one stride it is allowed)
    bwd = lambda x, dy, dx, add=None: H.op_layernorm_bwd(x, P, P, P, dy, 4, 8, dx, P, P, P, ws_bytes=1 << 20, add=add)
    refuses(H, bwd(P, Q, P), "in the place of")
    refuses(H, bwd(P, Q, Q), "in the place of")
    refuses(H, bwd(P, Q, Q, add=Q), "in the place of")
    refuses(H, H.op_layernorm_bwd(P, P, P, P, Q, 4, 8, W, P, P, P, ws_bytes=1 << 20, add=W, lddx=9), "in the place of")      # dx may be add with one stride only
    a = H.Mha(2, 4, 4, 2, 2, 8)
    p = [P + 4096 * i for i in range(9)]
    for i in range(3):
        refuses(H, H.op_mha_fwd(a, *p[:3], p[i]), "in the place of")
    for out in range(3):
        for other in [0, 1, 2, 3, 5] + [6 + j for j in range(3) if j != out]:
            t = list(p)
            t[6 + out] = p[other]
            refuses(H, H.op_mha_bwd(a, *t, ws=P + W, ws_bytes=1 << 30), "in the place of")


@pytest.mark.parametrize("version,says", [(11, "lacks pdae_"), (10, "ABI 10")])
def test_an_older_library_is_named_as_such(tmp_path, version, says):
    """Entry points were added without a new ABI number: a library of the number that lacks them is refused with what it lacks, not with an AttributeError later."""
    import os
    import subprocess
    import sys
    src, so = tmp_path / "old.c", tmp_path / "old.so"
    names = ["pdae_run_ops", "pdae_conv2d_wgrad_workspace_bytes", "pdae_gn_workspace_bytes"]
    src.write_text('const char* pdae_last_error(void) { return ""; }\nint pdae_abi_version(void) { return %d; }\n' % version + "".join(f"int {n}(void) {{ return 0; }}\n" for n in names))
    subprocess.run(["gcc", "-shared", "-fPIC", "-o", str(so), str(src)], check=True)
    r = subprocess.run([sys.executable, "-c", "from pdae_amd import hip\ntry:\n    hip.lib()\nexcept hip.PdaeError as e:\n    print('refused:', e)"], capture_output=True, text=True,
                       env=dict(os.environ, PDAE_HIP_LIB=str(so)), cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
    assert r.returncode == 0 and r.stdout.startswith("refused:") and says in r.stdout and str(so) in r.stdout, r.stdout + r.stderr[-600:]


def test_no_channels_are_refused_by_name(H):
    """The default scale of zero channels is no number: the refusal is the kernels' own, not a division by zero."""
    refuses(H, H.op_mha_fwd(H.Mha(2, 4, 4, 2, 1, 0), P, P, P, P), "head width 0")
