"""The bounds of paged_bounds.py, on the host: operands with all their terms are far within them, operands
that have lost one are not."""
import pytest

import paged_bounds as pb

torch = pytest.importorskip("torch")


def inputs(n, L, size, dense=False):
    g = torch.Generator().manual_seed(n)
    q = torch.randn((n, 4 * 128), generator=g) if dense else pb.sparse_queries(n, 4, 128, size, g)
    k = torch.randn((L, 4, 128), generator=g)
    k = (torch.round(k / k.abs().amax(-1, keepdim=True) * 127) / 127 * (1 if not dense else 3)).double()
    v = torch.randn((L, 4 * 128), generator=g) if dense else pb.sparse_values(L, 4, 128, g)
    return q.double().view(n, 4, 128), k, v.double().view(L, 4, 128), L - n, 128 ** -0.5


def worst(n, L, size, adds, dtype, q_terms, w_terms):
    a = inputs(n, L, size)
    o, S = pb.attend(*a)
    got, _ = pb.attend(*a, dtype, q_terms, w_terms)
    assert ((o != 0).sum((0, 1)) > 0).all()  # every column has a key that is seen
    r = ((got - o).abs() / o.abs().clamp_min(1e-300) / pb.bound(S, adds))[o != 0]
    assert (got[o == 0] == 0).all()
    return float(r.max())


@pytest.mark.parametrize("n,L,adds", [(40, 60, 16), (5, 100, 16), (300, 364, 28)])
def test_all_terms_are_within_the_bound_and_fewer_are_not(n, L, adds):
    for size in (6.4, 44.0):
        assert worst(n, L, size, adds, torch.float16, 2, 2) < 0.25
        assert worst(n, L, size, adds, torch.bfloat16, 3, 3) < 0.25
        assert worst(n, L, size, adds, torch.float16, 1, 2) > 10
        assert worst(n, L, size, adds, torch.float16, 2, 1) > 10
    assert worst(n, L, 44.0, adds, torch.bfloat16, 2, 3) > 1.2
    assert worst(n, L, 6.4, adds, torch.bfloat16, 3, 2) > 1.2


@pytest.mark.parametrize("n,L", [(40, 60), (5, 100), (300, 364)])
def test_dense_inputs_show_a_lost_binary16_term(n, L):
    a = inputs(n, L, 0, dense=True)
    o, _ = pb.attend(*a)
    size, _ = pb.attend(*a[:2], a[2].abs(), *a[3:])

    def rms(q_terms, w_terms):
        got, _ = pb.attend(*a, torch.float16, q_terms, w_terms)
        return float(((got - o) / size).square().mean().sqrt())

    assert rms(2, 2) < 0.05 * pb.DENSE_RMS
    assert rms(1, 2) > 2 * pb.DENSE_RMS and rms(2, 1) > 2 * pb.DENSE_RMS
