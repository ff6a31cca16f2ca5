"""The paged cache's attention where single numbers decide: infinities and NaN in places that are
seen or not, scores so large that their last place passes 1, values and queries at the ends of F32."""
import math

import pytest

import lai
import paged_ref as ref
from test_gpu_paged import DEV, Case, gen, i32

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


# ---- a value that is seen is not lost -----------------------------------------------------------
def poke(c, j, head, col, bad):
    """V of sequence 0's key j, as the cache holds it: a NaN's code in E4M3."""
    page = c.kv.v.shape[2]
    at = int(c.pages[0, j // page]), head, j % page, col
    if c.cache == torch.bfloat16:
        c.kv.v[at] = bad
    else:
        c.kv.v.view(torch.uint8)[at] = 0x7F


# one token or several; the part step at the end (its own value among it), whole steps, the first keys
# of a window and the one before it; and the kernel for many rows
SEEN = [(1, 37, 0, (5, 32, 36)), (1, 37, 20, (16, 17, 31, 36)), (1, 777, 0, (700, 768, 776)), (1, 130, 100, (29, 30, 128)),
        (3, 40, 0, (36, 37, 39)), (3, 100, 33, (64, 65, 70, 99)), (700, 800, 0, (99, 101, 500, 799)), (700, 837, 60, (70, 140, 836))]


@pytest.mark.parametrize("cache,bad", [("bf16", math.nan), ("bf16", math.inf), ("bf16", -math.inf), ("e4m3", math.nan)])
@pytest.mark.parametrize("dtype", list(ref.DTYPES))
@pytest.mark.parametrize("n,L,window,at", SEEN)
def test_a_value_that_is_seen_is_not_lost(n, L, window, at, cache, dtype, bad):
    for j in at:
        c = Case([n], [L], 4, 2, 128, cache, 16, dtype, seed=31)
        poke(c, j, 1, 77, bad)
        out = lai.paged_attention(c.q, c.kv, c.batch, window=window)
        pos = torch.arange(L - n, L, device=DEV)
        sees = (pos >= j) & (pos < j + (window or L))
        hit = torch.zeros((n, 4, 128), dtype=torch.bool, device=DEV)
        hit[sees, 2:, 77] = True
        hit = hit.view(n, -1)
        assert not torch.isfinite(out[hit]).any(), j
        o, tol = c.expected(window=window)  # (it leaves non-finite values out)
        assert ((out.double() - o).abs() <= tol)[~hit].all(), j


@pytest.mark.parametrize("n", [1, 3, 900])
@pytest.mark.parametrize("dtype", list(ref.DTYPES))
def test_a_value_that_is_seen_beside_a_missing_page_is_not_lost(n, dtype):
    L = n + 63
    c = Case([n], [L], 4, 2, 128, "e4m3", 16, dtype, seed=32)
    poke(c, 20, 1, 77, math.nan)
    pages = c.batch.pages.clone()
    pages[0, 0] = -1
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    out = lai.paged_attention(c.q, c.kv, lai.PagedBatch(c.batch.q_start, c.batch.kv_len, pages), err=err).view(n, 4, 128)
    assert int(err) == lai.LAI_DEVERR_PAGE
    assert torch.isnan(out[:, 2:, 77]).all()
    out[:, 2:, 77] = 0
    assert torch.isfinite(out).all()


# ---- scores whose last place is 2, 4, 8 .. -----------------------------------------------------
@pytest.mark.parametrize("n,L", [(1, 20000), (1100, 3000)])
@pytest.mark.parametrize("cache", list(ref.FORMATS))
@pytest.mark.parametrize("dtype", list(ref.DTYPES))
def test_equal_scores_of_any_magnitude_weigh_the_same(n, L, cache, dtype):
    """Every key is the same, so a row is the mean of what it sees. Tolerance: half a step of a BF16
    weight (2^-8; the means of |v| below 1, the result's own rounding as much again), and 2e-5 with
    F32, as for other rows of equal scores."""
    c = Case([n], [L], 2, 1, 64, cache, 64, dtype, seed=33)
    v = ref.sequence(ref.values(c.kv.v, c.kv.v_scale), c.pages[0], L)[:, 0]
    want = v.cumsum(0)[L - n:] / torch.arange(L - n + 1, L + 1, device=DEV)[:, None]
    tol = 2e-5 if dtype == "f32" else 2.0 ** -6
    for e in (9.3, 11.1, 13.7, 15.2, 20.2, 22.9, 23.9, 24.1, 24.5, 24.9, 25.3, 25.7, 26.2, 26.6, 27.1, 27.8, 28.4, 29.5, 33.0):
        for sign in (1, -1):
            k, q = torch.zeros_like(c.k_rows), torch.zeros_like(c.q)
            k[:, 0] = sign * 2.0 ** (e / 2)
            q[:, 0] = q[:, 64] = 2.0 ** (e / 2)
            lai.paged_kv_append(c.kv, c.whole, k, c.v_rows)
            out = lai.paged_attention(q, c.kv, c.batch, scale=1.0).double().view(n, 2, 64)
            assert (out - want[:, None]).abs().max() <= tol, (e, sign)


# ---- values of very different sizes --------------------------------------------------------------
def joint(c, s, L, dtype, cache, window=0):
    """(o, tolerance) of one sequence: as paged_ref.tolerance, but what a weight's last binary16 place
    is worth goes by the largest product of a weight and its value, among the keys the row sees."""
    n, H, hd = c.new[s], c.H, c.hd
    k = ref.sequence(ref.values(c.kv.k, c.kv.k_scale), c.pages[s], L)
    v = ref.sequence(ref.values(c.kv.v, c.kv.v_scale), c.pages[s], L)
    q = c.q[sum(c.new[:s]):sum(c.new[:s + 1])].double().view(n, H, hd)
    o, a, b, _ = ref.attend(q, k, v, L - n, hd ** -0.5, window)
    G = H // c.Hkv
    kh, vtop = k.repeat_interleave(G, 1), v.abs().amax(-1).repeat_interleave(G, 1)  # [keys, H]
    j, p = torch.arange(L, device=DEV), torch.arange(L - n, L, device=DEV)[:, None]
    see = (j <= p) & (j > p - (window or 1 << 40))
    w = torch.softmax((torch.einsum("nhd,khd->hnk", q, kh) * hd ** -0.5).masked_fill(~see, -math.inf), -1)
    u = (see.sum(-1)[None] * (w * vtop.T[:, None]).amax(-1)).T[..., None]
    return o.flatten(1), ref.tolerance(o, a, b, u, c.dtype, c.cache).flatten(1)


@pytest.mark.parametrize("n", [6, 1100])
@pytest.mark.parametrize("cache", ["i8", "e4m3"])
@pytest.mark.parametrize("dtype", list(ref.DTYPES))
@pytest.mark.parametrize("power", [24, 30, 42, 60, 100])
def test_a_large_value_reaches_only_who_sees_it(n, cache, dtype, power):
    L = n + 30
    c = Case([n], [L], 4, 2, 128, cache, 16, dtype, seed=34)
    j = 30 + n // 2
    v = c.v_rows.clone()
    v[j] *= 2.0 ** power
    lai.paged_kv_append(c.kv, c.whole, c.k_rows, v)
    out = lai.paged_attention(c.q, c.kv, c.batch).double()
    o, tol = joint(c, 0, L, dtype, cache)
    assert ((out - o).abs() <= tol).all()


@pytest.mark.parametrize("n", [1, 6, 1100])
@pytest.mark.parametrize("cache", ["i8", "e4m3"])
@pytest.mark.parametrize("dtype", list(ref.DTYPES))
@pytest.mark.parametrize("q_std", [1.0, 30.0])
def test_values_over_many_orders_lose_no_more_than_their_share(n, cache, dtype, q_std):
    """Value rows from 2^-45 to 2^45, under weights from 1 to e^-100 (q_std 30): a large value under a
    small weight takes nothing from a small value under a large one, but what it adds itself."""
    L = n + 300
    c = Case([n], [L], 2, 1, 64, cache, 16, dtype, seed=35, q_std=q_std)
    v = c.v_rows * torch.exp2(torch.randint(-45, 46, (L, 1), generator=gen(6), device=DEV).float())
    lai.paged_kv_append(c.kv, c.whole, c.k_rows, v)
    out = lai.paged_attention(c.q, c.kv, c.batch).double()
    o, tol = joint(c, 0, L, dtype, cache)
    assert ((out - o).abs() <= tol).all()


@pytest.mark.parametrize("n", [1, 6, 1100])
@pytest.mark.parametrize("cache", ["i8", "e4m3"])
@pytest.mark.parametrize("dtype", list(ref.DTYPES))
@pytest.mark.parametrize("power", [-80, -50, 70, 110])
def test_values_of_one_extreme_size(n, cache, dtype, power):
    c = Case([n], [n + 50], 2, 1, 64, cache, 16, dtype, seed=36)
    lai.paged_kv_append(c.kv, c.whole, c.k_rows, c.v_rows * 2.0 ** power)
    out = lai.paged_attention(c.q, c.kv, c.batch).double()
    o, tol = joint(c, 0, n + 50, dtype, cache)
    assert ((out - o).abs() <= tol).all()


@pytest.mark.parametrize("n", [1, 6, 1100])
@pytest.mark.parametrize("cache", list(ref.FORMATS))
@pytest.mark.parametrize("dtype", list(ref.DTYPES))
@pytest.mark.parametrize("slope", [0.02, 0.3])
def test_scores_that_rise_along_the_sequence(n, cache, dtype, slope):
    """The maximum moves at every step, by little or much, while the values shrink."""
    L = n + 900
    c = Case([n], [L], 2, 1, 64, cache, 16, dtype, seed=38)
    at = torch.arange(L, device=DEV)[:, None]
    k = torch.zeros_like(c.k_rows)
    k[:, :1] = slope * at
    lai.paged_kv_append(c.kv, c.whole, k, c.v_rows * torch.exp2(-0.01 * at))
    c.q.zero_()
    c.q[:, 0], c.q[:, 64] = 8.0, -8.0
    out = lai.paged_attention(c.q, c.kv, c.batch).double()
    o, tol = joint(c, 0, L, dtype, cache)
    assert ((out - o).abs() <= tol).all()


@pytest.mark.parametrize("n", [6, 1100])
@pytest.mark.parametrize("cache", ["i8", "e4m3"])
@pytest.mark.parametrize("dtype", list(ref.DTYPES))
def test_value_scales_that_append_never_makes(n, cache, dtype):
    """A cache filled by other means: scales that are zero, negative or below F32's normal range."""
    L = n + 100
    c = Case([n], [L], 4, 2, 128, cache, 16, dtype, seed=39)
    s = c.kv.v_scale
    pick = torch.randint(0, 8, s.shape, generator=gen(7), device=DEV)
    s.copy_(torch.where(pick == 0, 0.0, torch.where(pick == 1, -s, torch.where(pick == 2, s * 1e-38, s))))
    c.check()


# ---- queries and keys at the ends of F32 ----------------------------------------------------------
# (key scales end at 2^90: behind that only the kernel for few rows has the room)
@pytest.mark.parametrize("n,power", [(n, p) for n in (1, 6) for p in (90, 105, 112, 114, 118, -90, -110)] +
                         [(1100, p) for p in (60, 94, -90, -110)])
@pytest.mark.parametrize("cache", ["i8", "e4m3"])
@pytest.mark.parametrize("dtype", list(ref.DTYPES))
def test_small_queries_over_large_keys(n, power, cache, dtype):
    c = Case([n], [n + 50], 2, 1, 64, cache, 16, dtype, seed=37)
    lai.paged_kv_append(c.kv, c.whole, c.k_rows * 2.0 ** power, c.v_rows)
    c.q *= 2.0 ** -power
    c.check()


# ---- tensors that a call makes ---------------------------------------------------------------------
@pytest.mark.parametrize("new,keys", [([1, 1], [20000, 900]), ([300], [9000])])
def test_calls_on_a_stream_beside_a_busy_current_one(new, keys):
    """Scratch and outputs that the call makes itself, while the current stream is far behind and goes
    on making and dropping memory of the same sizes."""
    c = Case(new, keys, 8, 4, 128, "i8", 64, "f32", seed=40)
    want = c.check()
    k, v = lai.paged_kv_read(c.kv, c.whole, sum(keys), torch.float32)
    x = torch.randn((8192, 8192), device=DEV, dtype=torch.bfloat16)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    outs = []
    for _ in range(20):
        x = x @ x  # about a millisecond each
        stale = torch.full((10_000_000,), 7.0, device=DEV)
        del stale
        outs.append(lai.paged_attention(c.q, c.kv, c.batch, stream=stream))
        outs.append(lai.paged_kv_read(c.kv, c.whole, sum(keys), torch.float32, stream=stream))
    stream.synchronize()
    for got in outs:
        if isinstance(got, tuple):
            assert torch.equal(got[0], k) and torch.equal(got[1], v)
        else:
            assert torch.equal(got, want)


# ---- batches that are not well formed ---------------------------------------------------------------
@pytest.mark.parametrize("many", [1, 8])
@pytest.mark.parametrize("cache,dtype", [("i8", "f32"), ("bf16", "bf16")])
def test_a_malformed_batch_leaves_the_scratch_as_it_was(many, cache, dtype):
    """q_start that decreases, or leaves the rows by little or by all an int has: flagged, and the next
    call with the same scratch is right."""
    import random
    r = random.Random(many)
    rows, keys = 200 * many, [r.randint(100, 3000) + 200 * many for _ in range(10)]
    c = Case([20 * many] * 10, keys, 4, 2, 128, cache, 16, dtype, seed=41)
    scratch = lai.paged_attention_scratch(128)
    want = c.check(scratch=scratch)
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    out = torch.empty_like(c.q)
    bad = [[x * many for x in (0, 76, 12, 96, 192, 154, 176, 72, 44, 43, 112)]]
    bad += [[0] + [r.randint(0, rows) for _ in range(10)] for _ in range(60)]
    bad += [sorted(r.choice([-2 ** 31, -5, 0, 3, rows // 2, rows, rows + 1, 2 ** 27, 2 ** 28, 2 ** 31 - 1]) for _ in range(11))
            for _ in range(60)]
    for q_start in bad:
        assert len(q_start) == 11
        fine = all(0 <= a <= b <= rows for a, b in zip(q_start, q_start[1:]))
        err.zero_()
        lai.paged_attention(c.q, c.kv, lai.PagedBatch(i32(q_start), c.batch.kv_len, c.batch.pages), scratch=scratch, out=out, err=err)
        assert (int(err) != 0) != fine, q_start
        assert not scratch[:1024].view(torch.int32).any(), q_start
    assert torch.equal(c.check(scratch=scratch), want)


@pytest.mark.parametrize("n", [3, 400])
def test_sequences_beside_one_that_leaves_the_rows_are_computed(n):
    c = Case([n, n, n], [n + 60, n + 700, n + 9], 4, 2, 64, "i8", 16, "f32", seed=42)
    want = c.check()
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    for q_start, good in (([0, n, 2 * n, 3 * n + 1], (0, 1)), ([0, n, 2 * n, 2 ** 31 - 1], (0, 1)), ([-7, n, 2 * n, 3 * n], (1, 2)),
                          ([-2 ** 31, n, 2 * n, 2 ** 31 - 1], (1,))):
        out = torch.full_like(c.q, 9.0)
        err.zero_()
        lai.paged_attention(c.q, c.kv, lai.PagedBatch(i32(q_start), c.batch.kv_len, c.batch.pages), out=out, err=err)
        assert int(err) == lai.LAI_DEVERR_POSITION
        for s in range(3):
            got = out[s * n:(s + 1) * n]
            if s in good:  # (the schedule differs, so the bits may)
                assert (got - want[s * n:(s + 1) * n]).abs().max() <= 2e-5
            else:
                assert (got == 9).all()
