"""F32 queries over the paged cache against the bounds of paged_bounds.py, which no lost term passes."""
import pytest

import lai
import paged_bounds as pb
import paged_ref as ref
from test_gpu_paged import DEV, Case, gen

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
# few rows: a lane adds 8 weights a step, lanes and warps join; many rows: 16 pairs a block, 3 blocks
SHAPES = [([1], [40], 16), ([1] * 20, [60] * 20, 16), ([5], [100], 16), ([1, 2], [333, 70], 24), ([300], [364], 28),
          ([150, 160], [200, 160], 28)]


def sequences(c):
    kd, vd = ref.values(c.kv.k, c.kv.k_scale), ref.values(c.kv.v, c.kv.v_scale)
    at, G = 0, c.H // c.Hkv
    for s, (n, L) in enumerate(zip(c.new, c.keys)):
        k, v = (ref.sequence(x, c.pages[s], L).repeat_interleave(G, 1) for x in (kd, vd))
        yield slice(at, at + n), c.q[at:at + n].double().view(n, c.H, c.hd), k, v, L - n
        at += n


@pytest.mark.parametrize("size", [6.4, 44.0])
@pytest.mark.parametrize("cache", list(ref.FORMATS))
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("new,keys,adds", SHAPES)
def test_every_term_of_every_element(new, keys, adds, hd, cache, size):
    c = Case(new, keys, 8, 4, hd, cache, 16, "f32", seed=51)
    g = gen(52)
    c.q = pb.sparse_queries(sum(new), 8, hd, size * (hd / 128) ** 0.5, g, DEV)
    k = torch.randn(c.k_rows.shape, generator=g, device=DEV).view(-1, 4, hd)
    k = (k / k.abs().amax(-1, keepdim=True)).flatten(1)
    v = torch.cat([pb.sparse_values(L, 4, hd, g, DEV) for L in keys])
    lai.paged_kv_append(c.kv, c.whole, k, v)
    out = c_out(c)
    for rows, q, kd, vd, pos0 in sequences(c):
        o, S = pb.attend(q, kd, vd, pos0, hd ** -0.5)
        got = out[rows].double().view(o.shape)
        assert (got[o == 0] == 0).all()
        worst = ((got - o).abs() / o.abs().clamp_min(1e-300) / pb.bound(S, adds))[o != 0].max()
        assert worst <= 1, float(worst)


@pytest.mark.parametrize("cache", list(ref.FORMATS))
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("new,keys", [(n, k) for n, k, _ in SHAPES])
def test_dense_inputs(new, keys, hd, cache):
    c = Case(new, keys, 8, 4, hd, cache, 16, "f32", seed=53)
    out = c_out(c)
    for rows, q, kd, vd, pos0 in sequences(c):
        o, _ = pb.attend(q, kd, vd, pos0, hd ** -0.5)
        a, _ = pb.attend(q, kd, vd.abs(), pos0, hd ** -0.5)
        rms = ((out[rows].double().view(o.shape) - o) / a.clamp_min(1e-300)).square().mean().sqrt()
        assert rms <= pb.DENSE_RMS, float(rms)


def c_out(c):
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    out = lai.paged_attention(c.q, c.kv, c.batch, err=err)
    assert int(err) == 0
    return out
