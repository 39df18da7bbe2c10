"""Calls that the token operators' documentation allows, as far as their checks on the host go: no kernel is launched here."""
import ctypes as C

import pytest

from panogrf_amd._lib import lib
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
