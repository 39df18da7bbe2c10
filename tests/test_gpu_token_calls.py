"""Calls of the token operators that their documentation allows, at the edges of what they took (HIP)."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_one_query_a_stream_in_sequence_first_memory():
    """[1, B, H, 2, d].transpose(0, 1): contiguous, with over 2^22 values from the only token to the next."""
    from panogrf_amd.attention import diff_attention, diff_attention_cached
    g = torch.Generator(device='cuda').manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=g, device='cuda').bfloat16()
    B, H, Hk, D, M = 520, 32, 8, 128, 5
    q = r(1, B, H, 2, D).transpose(0, 1)
    assert q.stride(1) > 1 << 22 and q.is_contiguous()
    k, v, lam, do = r(B, M, Hk, 2, D), r(B, M, Hk, 2 * D), torch.rand(H, generator=g, device='cuda'), r(B, 1, H, 2 * D)
    n = torch.arange(B, device='cuda', dtype=torch.int32) % (M + 1)

    def run(q, k, v):
        ts = [t.detach().requires_grad_(True) for t in (q, k, v, lam)]
        out = diff_attention(*ts)
        return (out.detach(), *torch.autograd.grad(out, ts, do), diff_attention_cached(q, k, v, lam, n))
    one = torch.empty(B * H * 2 * D, device='cuda', dtype=torch.bfloat16).view(B, 1, H, 2, D).copy_(q)
    assert one.stride(1) < 1 << 22
    assert all(torch.equal(a, b) for a, b in zip(run(q, k, v), run(one, k, v)))
    # keys of one token likewise
    k1, v1 = k[:, :1].contiguous().transpose(0, 1).contiguous().transpose(0, 1), r(1, B, 32, 2 * D).transpose(0, 1)[:, :, ::4]
    far = v1.as_strided(v1.shape, (v1.stride(0), 1 << 23, v1.stride(2), 1))
    n.clamp_(max=1)
    assert all(torch.equal(a, b) for a, b in zip(run(q, k1, far), run(one, k[:, :1].clone(), v1.clone(memory_format=torch.contiguous_format))))
