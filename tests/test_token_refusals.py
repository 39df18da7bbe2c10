"""What the token operators refuse, on the host: no kernel is launched here."""
import ctypes as C

import pytest
import torch

from panogrf_amd._lib import PgrfError, lib

PTR = 1 << 20        # an address no kernel ever sees: every call below ends in the checks before it


def norm_c(dtype=0, rows=4, channels=8, flags=6, rpg=4, x=PTR, y=PTR, gate=None, x_out=PTR, z=PTR, stats=None):
    from panogrf_amd._lib import PgrfBlockNorm
    a = PgrfBlockNorm(x=x, y=y, gate=gate, x_out=x_out, z_out=z, stats=stats, rows=rows, rows_per_gate=rpg, dtype=dtype, C=channels, flags=flags, scale=1.0, eps=1e-6)
    return lib.pgrf_block_norm(C.byref(a), None)


def test_packed_structures_are_the_header_s():
    from panogrf_amd import _lib, _token
    for packed, fields in ((_token.BLOCK_NORM, _lib.PgrfBlockNorm), (_token.ROTARY, _lib.PgrfRotary), (_token.DIFF_ATTN, _lib.PgrfDiffAttn)):
        assert packed.size == C.sizeof(fields)
        marks = []
        for i, (n, t) in enumerate(fields._fields_):
            marks.append(t(i + 1).value)
        got = fields.from_buffer_copy(packed.pack(*marks))
        assert [getattr(got, n) for n, _ in fields._fields_] == marks


@pytest.mark.parametrize('kw,code', [(dict(dtype=3), -3), (dict(dtype=-1), -3), (dict(channels=0), -3), (dict(channels=8193), -3), (dict(rows=-1), -1),
                                     (dict(flags=8), -1), (dict(y=None), -1), (dict(y=None, flags=0), -1), (dict(gate=PTR, rpg=3), -1), (dict(gate=PTR, rpg=0), -1),
                                     (dict(x=None), -1), (dict(x_out=None), -1), (dict(z=None), -1), (dict(stats=PTR + 4), -1)])
def test_block_norm_entry(kw, code):
    assert norm_c(**kw) == code and b'pgrf_block_norm' in lib.pgrf_last_error()


def test_block_norm_entries_without_rows():
    assert norm_c(rows=0) == 0
    n = lib.pgrf_block_norm_backward_workspace_bytes(100, 64, 10)
    assert n >= 64 * 5 * 4
    from panogrf_amd._lib import PgrfBlockNorm

    def back(**kw):
        a = PgrfBlockNorm(**{**dict(x=PTR, y=PTR, gate=PTR, stats=PTR, dx_out=PTR, dz=PTR, dx=PTR, dy=PTR, dgate=PTR, dpost_w=PTR, dpre_w=PTR, rows=100, rows_per_gate=10,
                                    dtype=0, C=64, flags=6, scale=1.0), **kw})
        return lib.pgrf_block_norm_backward(C.byref(a), None)
    assert back() == -1 and b'workspace' in lib.pgrf_last_error()
    assert back(workspace=PTR, workspace_bytes=64) == -1 and b'workspace' in lib.pgrf_last_error()
    assert back(gate=None) == -1 and b'dgate' in lib.pgrf_last_error()
    assert back(stats=None) == back(x=None) == back(rows_per_gate=7) == -1
    assert back(rows=200000, rows_per_gate=2, workspace=PTR, workspace_bytes=1 << 40) == -3
    assert lib.pgrf_block_norm(None, None) == lib.pgrf_block_norm_backward(None, None) == lib.pgrf_rotary(None, None) == -1


@pytest.mark.parametrize('kw', [dict(y=torch.zeros(2, 3, 7)), dict(gate=torch.ones(8)), dict(y=torch.zeros(2, 3, 8), gate=torch.ones(3, 8)),
                                dict(y=torch.zeros(2, 3, 8), gate=torch.ones(7)), dict(kind='group'), dict(post_weight=torch.ones(8)), dict(pre=False),
                                dict(pre_weight=torch.ones(7)), dict(pre_bias=torch.ones(8)), dict(y=torch.zeros(2, 3, 8).half()),
                                dict(y=torch.zeros(2, 3, 8), post=False, post_weight=torch.ones(8)), dict()])
def test_block_norm(kw):
    from panogrf_amd.block_norm import block_norm
    with pytest.raises(PgrfError):          # (the last: a CPU tensor)
        block_norm(torch.zeros(2, 3, 8), **kw)


def test_block_norm_types():
    from panogrf_amd.block_norm import block_norm
    for x in (torch.zeros(2, 8).double(), torch.zeros(2, 8).int(), torch.zeros(()), torch.zeros(2, 8193), torch.zeros(2, 0), None):
        with pytest.raises(PgrfError):
            block_norm(x)


@pytest.mark.parametrize('kw,code', [(dict(dtype=5), -3), (dict(D=1), -1), (dict(rot=3), -3), (dict(rot=0), -3), (dict(rot=18), -3), (dict(D=512, rot=258), -3),
                                     (dict(hq=0), -1), (dict(hk=-1), -1), (dict(kind=4), -1), (dict(base=0.0), -1), (dict(base=float('nan')), -1),
                                     (dict(scaling=4), -1), (dict(scaling=1, factor=0.0), -1), (dict(scaling=2, rot=2, factor=2.0), -3),
                                     (dict(scaling=3, factor=2.0, low=4.0, high=4.0), -1), (dict(q=None), -1), (dict(hk=1, k=None), -1), (dict(hq=1 << 17), -3)])
def test_rotary_entry(kw, code):
    a = dict(q=PTR, hq=1, k=PTR, hk=0, kind=0, dtype=0, D=16, rot=16, base=1e4, scaling=0, factor=1.0, low=1.0, high=32.0)
    a.update(kw)
    from panogrf_amd._lib import PgrfRotary
    r = PgrfRotary(q=a['q'], k=a['k'], positions=PTR, q_out=PTR, k_out=PTR, q_sb=16, q_sn=16, q_sh=16, k_sb=16, k_sn=16, k_sh=16, base=a['base'], factor=a['factor'],
                   trained_length=4096.0, low=a['low'], high=a['high'], dtype=a['dtype'], B=2, N=3, D=a['D'], q_heads=a['hq'], k_heads=a['hk'], rotary_dim=a['rot'],
                   position_type=a['kind'], scaling=a['scaling'], magnitude=1.0)
    rc = lib.pgrf_rotary(C.byref(r), None)
    assert rc == code and b'pgrf_rotary' in lib.pgrf_last_error()


@pytest.mark.parametrize('kw', [dict(rotary_dim=3), dict(rotary_dim=18), dict(rotary_dim=0), dict(layout='quarter'), dict(scaling='cubic'),
                                dict(positions=torch.arange(4)), dict(positions=torch.arange(3).half()), dict(positions=torch.zeros(3, 3)), dict(positions=None),
                                dict(k=torch.zeros(2, 4, 1, 16)), dict(k=torch.zeros(2, 3, 1, 8)), dict(k=torch.zeros(2, 3, 1, 16).half()),
                                dict(k=torch.zeros(2, 3, 0, 16)), dict()])
def test_rotary(kw):
    from panogrf_amd.rotary import rotary
    kw = dict(k=None, positions=torch.arange(3)) | kw
    with pytest.raises(PgrfError):          # (the last: a CPU tensor)
        rotary(torch.zeros(2, 3, 4, 16), kw.pop('k'), kw.pop('positions'), **kw)


def test_rotary_positions_have_no_gradient():
    from panogrf_amd.rotary import rotary
    with pytest.raises(PgrfError, match='detach'):
        rotary(torch.zeros(2, 3, 4, 16), None, torch.zeros(3, requires_grad=True))


def attn(**kw):
    from panogrf_amd._lib import PgrfDiffAttn
    a = PgrfDiffAttn(q=PTR, k=PTR, v=PTR, lam=PTR, out=PTR, dtype=1, B=2, N=3, M=4, H=4, Hk=2, D=64, scale=0.1)
    for n in ('q_sb', 'q_sn', 'q_sh', 'q_sm', 'k_sb', 'k_sn', 'k_sh', 'k_sm', 'v_sb', 'v_sn', 'v_sh'):
        setattr(a, n, 64)
    for n, x in kw.items():
        setattr(a, n, x)
    return a


BAD = [(dict(dtype=3), -3), (dict(D=48), -3), (dict(D=256), -3), (dict(M=0), -1), (dict(H=3), -1), (dict(Hk=0), -1), (dict(N=-1), -1), (dict(scale=0.0), -1),
       (dict(scale=-1.0), -1), (dict(scale=float('nan')), -1), (dict(q=None), -1), (dict(v=None), -1), (dict(lam=None), -1), (dict(q=PTR + 8), -1),
       (dict(k_sn=63), -1), (dict(q_sm=4), -1), (dict(maps_out=PTR), -1), (dict(N=1 << 30), -3)]


@pytest.mark.parametrize('kw,code', BAD + [(dict(out=None), -1), (dict(N=1, M=100000, B=1), -1)])       # (the last: a cut key axis without a workspace)
def test_diff_attention_entry(kw, code):
    assert lib.pgrf_diff_attention(C.byref(attn(**kw)), None) == code and b'pgrf_diff_attention' in lib.pgrf_last_error()


@pytest.mark.parametrize('kw,code', [b for b in BAD if 'maps_out' not in b[0]] + [(dict(lse=None, maps_out=None), -1), (dict(lse=None), -1), (dict(lengths=PTR), -3), (dict(B=0), -1)])
def test_diff_attention_backward_entry(kw, code):
    a = attn(**{**dict(lse=PTR, maps_out=PTR), **kw})
    assert lib.pgrf_diff_attention_backward(C.byref(a), PTR, PTR, PTR, PTR, PTR, None) == code


def test_diff_attention_backward_arguments():
    a = attn(lse=PTR, maps_out=PTR)
    assert lib.pgrf_diff_attention_backward(C.byref(a), PTR, PTR, PTR, None, PTR, None) == -1          # dk without dv
    assert lib.pgrf_diff_attention_backward(C.byref(a), None, PTR, PTR, PTR, PTR, None) == -1
    assert lib.pgrf_diff_attention_backward(C.byref(a), PTR, PTR, PTR, PTR, PTR, None) == -1 and b'workspace' in lib.pgrf_last_error()
    assert lib.pgrf_diff_attention(None, None) == -1
    assert lib.pgrf_diff_attention(C.byref(attn(B=0)), None) == 0


Q, K, V, L = torch.zeros(2, 3, 4, 2, 32), torch.zeros(2, 5, 2, 2, 32), torch.zeros(2, 5, 2, 64), torch.zeros(4)


@pytest.mark.parametrize('a,kw', [((Q[..., :24], K, V, L), {}), ((Q, K[..., :16], V, L), {}), ((Q, K, V[..., :32], L), {}), ((Q, K, V, L[:3]), {}), ((Q, K[:, :4], V, L), {}),
                                  ((Q, K[:1], V, L), {}), ((Q[:, :, :3], K, V, L[:3]), {}), ((Q.half(), K, V, L), {}), ((Q.double(), K.double(), V.double(), L), {}),
                                  ((Q, K, V, L.half()), {}), ((Q, K, V, None), {}), ((Q.flatten(-2), K, V, L), {}), ((Q, K, V, L), dict(scale=0.0)),
                                  ((Q, K, V, L), dict(key_mask=torch.ones(2, 5))), ((Q, K, V, L), dict(key_mask=torch.ones(2, 4) > 0)),
                                  ((Q, K, V, L), dict(key_mask=torch.ones(2, 3, 5) > 0)), ((Q, K, V, L), {})])
def test_diff_attention(a, kw):
    from panogrf_amd.attention import diff_attention
    with pytest.raises(PgrfError):          # (the last: CPU tensors)
        diff_attention(*a, **kw)


@pytest.mark.parametrize('n', [torch.tensor([1, 2]), torch.tensor([1], dtype=torch.int32), None, torch.tensor([1.0, 2.0]), torch.tensor([1, 2], dtype=torch.int32)])
def test_diff_attention_cached(n):
    from panogrf_amd.attention import diff_attention_cached
    with pytest.raises(PgrfError):
        diff_attention_cached(Q, K, V, L, n)
    with pytest.raises(PgrfError, match='gradients|GPU|lengths'):
        diff_attention_cached(Q.requires_grad_(True), K, V, L, n)
    Q.requires_grad_(False)
