"""Calls that the token operators' documentation allows, as far as their checks on the host go: no kernel is launched here."""
import ctypes as C

import pytest
import torch

from panogrf_amd._lib import PgrfBlockNorm, PgrfRotary, lib
from tests.test_token_refusals import PTR, attn

FAR = 1 << 23


@pytest.mark.parametrize('kw', [dict(N=1, q_sn=FAR), dict(M=1, k_sn=FAR, v_sn=FAR), dict(N=1, q_sn=-64), dict(N=1, M=1, q_sn=FAR, k_sn=FAR, v_sn=FAR)])
def test_strides_of_axes_of_one_token_do_not_matter(kw):
    a = attn(**kw, lse=PTR)
    assert lib.pgrf_diff_attention_backward(C.byref(a), PTR, PTR, PTR, PTR, PTR, None) == -1 and b'workspace' in lib.pgrf_last_error()   # (what is asked behind strides)


@pytest.mark.parametrize('kw', [dict(N=2, q_sn=FAR), dict(M=2, k_sn=FAR), dict(M=2, v_sn=FAR), dict(N=1, q_sm=FAR), dict(k_sm=-64)])
def test_those_of_others_do(kw):
    a = attn(**kw, lse=PTR)
    assert lib.pgrf_diff_attention_backward(C.byref(a), PTR, PTR, PTR, PTR, PTR, None) == -3 and b'stride' in lib.pgrf_last_error()


def test_many_shared_gate_rows():
    """Only the gate's own gradient has a limit of them; without it they cost no workspace of their own either."""
    from panogrf_amd._lib import PgrfError
    from panogrf_amd.block_norm import block_norm
    x, gate = torch.zeros(60001, 2, 4), torch.ones(60001, 4)
    for grad in (False, True):
        with torch.set_grad_enabled(grad), pytest.raises(PgrfError, match='GPU'):         # (as far as CPU tensors go)
            block_norm(x.requires_grad_(grad), x.detach(), gate)
    with torch.no_grad(), pytest.raises(PgrfError, match='GPU'):
        block_norm(x, x, gate.requires_grad_(True))
    with pytest.raises(PgrfError, match='60000'):
        block_norm(x, x, gate)
    assert lib.pgrf_block_norm_backward_workspace_bytes(1 << 20, 64, 2) < 1 << 20
    assert lib.pgrf_block_norm_backward_workspace_bytes(60000 * 2, 64, 2) >= 60000 * 5 * 64 * 4
    a = PgrfBlockNorm(x=PTR, y=PTR, gate=PTR, stats=PTR, dx_out=PTR, dz=PTR, dx=PTR, dy=PTR, dpost_w=PTR, dpre_w=PTR, rows=1 << 20, rows_per_gate=2, dtype=0, C=64, flags=6,
                      scale=1.0, workspace=PTR, workspace_bytes=64)
    assert lib.pgrf_block_norm_backward(C.byref(a), None) == -1 and b'workspace' in lib.pgrf_last_error()


@pytest.mark.parametrize('dtype', [0, 1, 2])
@pytest.mark.parametrize('kw', [dict(B=524288, N=64, M=64, H=16, Hk=16, D=32), dict(B=1 << 20, N=1, M=3, H=16, Hk=16, D=64), dict(B=(1 << 22) - 1, N=1, M=1, H=8, Hk=8, D=128),
                                dict(B=(1 << 14) - 1, N=1 << 13, M=1, H=4, Hk=1, D=32), dict(B=1 << 18, N=65, M=33, H=31, Hk=31, D=128)])
def test_many_workgroups(kw, dtype):
    """B Hk below 2^25, B H N and B Hk M below 2^29: every launch has room for them."""
    a = attn(**kw, dtype=dtype, lse=PTR, workspace=PTR, workspace_bytes=16)
    assert lib.pgrf_diff_attention_backward(C.byref(a), PTR, PTR, PTR, PTR, PTR, None) == -1 and b'workspace' in lib.pgrf_last_error()   # (asked for behind the tiles)


def test_too_many_workgroups():
    a = attn(B=1 << 26, N=1, M=1, H=2, Hk=2, D=64, lse=PTR, workspace=PTR, workspace_bytes=1 << 62)
    assert lib.pgrf_diff_attention_backward(C.byref(a), PTR, PTR, PTR, PTR, PTR, None) == -3 and b'tiles' in lib.pgrf_last_error()
    assert lib.pgrf_diff_attention(C.byref(a), None) == -3 and b'tiles' in lib.pgrf_last_error()


def rotary(**kw):
    a = dict(q=PTR, positions=PTR, q_out=PTR, q_sb=0, q_sn=0, q_sh=0, base=1e4, factor=1.0, dtype=1, q_heads=1, rotary_dim=2, magnitude=1.0)
    return lib.pgrf_rotary(C.byref(PgrfRotary(**{**a, **kw})), None)


def test_rotary_tokens():
    """What no launch holds is refused as such, not by the runtime: 2^30 tokens (less where over 2^21 values and pairs of a workgroup's tokens would have to be counted)."""
    for kw in (dict(B=1 << 15, N=(1 << 15) + 1, D=2), dict(B=1 << 15, N=1 << 12, D=33, q_heads=31 * 1024)):
        assert rotary(**kw) == -3 and b'too many tokens' in lib.pgrf_last_error()
