"""The token operators have no forward-mode derivatives and say so: an output without a tangent would be a derivative of zero.  On the host; no kernel is launched."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

from panogrf_amd._lib import PgrfError

X, W = torch.zeros(2, 3, 32), torch.ones(32)
Q, K, V, L = torch.zeros(2, 3, 4, 2, 32), torch.zeros(2, 5, 2, 2, 32), torch.zeros(2, 5, 2, 64), torch.zeros(4)
P = torch.zeros(3)


def calls():
    from panogrf_amd.attention import diff_attention, diff_attention_cached
    from panogrf_amd.block_norm import block_norm
    from panogrf_amd.rotary import rotary
    n = torch.tensor([1, 2], dtype=torch.int32)
    return {'block_norm': (lambda x, y, g, w, v: block_norm(x, y, g, post_weight=w, pre_weight=v), (X, X.clone(), W.clone(), W, W.clone())),
            'block_norm alone': (lambda x, b: block_norm(x, pre_bias=b, kind='layer'), (X, W)),
            'rotary': (rotary, (X.view(2, 3, 2, 16), X.view(2, 3, 2, 16).clone(), P)),
            'rotary of one': (lambda q, p: rotary(q, None, p), (X, P)),
            'diff_attention': (diff_attention, (Q, K, V, L)),
            'diff_attention_cached': (lambda *a: diff_attention_cached(*a, n), (Q, K, V, L))}


@pytest.mark.parametrize('name', ['block_norm', 'block_norm alone', 'rotary', 'rotary of one', 'diff_attention', 'diff_attention_cached'])
@pytest.mark.parametrize('asks', [False, True])
def test_tangents_are_refused(name, asks):
    call, args = calls()[name]
    for i in range(len(args)):
        with fwd.dual_level():
            # (another argument that asks for a gradient makes no difference)
            given = [fwd.make_dual(t, torch.ones_like(t)) if j == i else t.clone().requires_grad_(asks and t is not P and 'cached' not in name) for j, t in enumerate(args)]
            with pytest.raises(PgrfError, match='forward'):
                call(*given)
            with torch.no_grad(), pytest.raises(PgrfError, match='forward'):
                call(*given)
        with pytest.raises(PgrfError, match='forward'):
            torch.func.jvp(lambda t: call(*[t if j == i else u for j, u in enumerate(args)]), (args[i],), (torch.ones_like(args[i]),))


@pytest.mark.parametrize('name', ['block_norm', 'rotary', 'diff_attention', 'diff_attention_cached'])
def test_a_level_without_tangents_is_not(name):
    call, args = calls()[name]
    with fwd.dual_level(), pytest.raises(PgrfError, match='GPU'):        # (as far as CPU tensors go)
        call(*args)


def test_upstream_gradients_with_tangents_are_refused():
    from panogrf_amd._token import first_derivatives_only
    backward = first_derivatives_only(lambda ctx, *g: g)
    with fwd.dual_level():
        assert backward(None, X, None)[0] is X
        for enabled in (False, True):
            with torch.set_grad_enabled(enabled), pytest.raises(PgrfError, match='forward'):
                backward(None, None, fwd.make_dual(X, X + 1))
