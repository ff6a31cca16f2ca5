"""The paged key/value cache (append, read back) and the attention over it, against their
definitions in 64 bits (paged_ref.py)."""
import math

import pytest

import lai
import paged_ref as ref

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
DEV = "cuda"


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def starts(new):
    return i32([0]).new_tensor([sum(new[:i]) for i in range(len(new) + 1)])


class Case:
    """A pool filled with random keys and values, a ragged batch over it and its query rows.
    pos0s / lens as the batch gives them; garbage: what unused places hold."""

    def __init__(self, new, keys, H, Hkv, hd, cache, page, dtype, seed=0, garbage=None, q_std=1.0):
        self.new, self.keys, self.H, self.Hkv, self.hd = new, keys, H, Hkv, hd
        self.cache, self.dtype = ref.FORMATS[cache], ref.DTYPES[dtype]
        g = gen(seed)
        pages, pool = ref.make_pages(keys, page, seed=seed)
        self.kv = lai.PagedKV.allocate(pool, Hkv, page, hd, self.cache)
        self.pages = pages
        self.k_rows = torch.randn((sum(keys), Hkv * hd), generator=g, device=DEV)
        self.v_rows = torch.randn((sum(keys), Hkv * hd), generator=g, device=DEV)
        self.whole = lai.PagedBatch(starts(keys), i32(keys), pages.to(DEV))
        err = torch.zeros(1, dtype=torch.int32, device=DEV)
        if garbage is not None:
            for t in (self.kv.k, self.kv.v):
                if self.cache == torch.bfloat16:
                    t.fill_(garbage)
                elif self.cache == torch.float8_e4m3fn:
                    t.view(torch.uint8).fill_(0x7F)
            for t in (self.kv.k_scale, self.kv.v_scale):
                if t is not None:
                    t.fill_(garbage)
        if sum(keys):
            lai.paged_kv_append(self.kv, self.whole, self.k_rows, self.v_rows, err=err)
        assert int(err) == 0
        self.batch = lai.PagedBatch(starts(new), i32(keys), pages.to(DEV))
        self.q = (torch.randn((sum(new), H * hd), generator=g, device=DEV) * q_std).to(self.dtype)

    def expected(self, scale=None, window=0):
        """(o, tolerance) in float64, rows in order."""
        scale = self.hd ** -0.5 if scale is None else scale
        kd = ref.values(self.kv.k, self.kv.k_scale)
        vd = ref.values(self.kv.v, self.kv.v_scale)
        os, tols, at = [], [], 0
        for s, (n, L) in enumerate(zip(self.new, self.keys)):
            q = self.q[at:at + n].double().view(n, self.H, self.hd)
            at += n
            o, a, b, u = ref.attend(q, ref.sequence(kd, self.pages[s], L),
                                 ref.sequence(vd, self.pages[s], L), L - n, scale, window)
            os.append(o.flatten(1))
            tols.append(ref.tolerance(o, a, b, u, self.dtype, self.cache).flatten(1))
        return torch.cat(os), torch.cat(tols)

    def check(self, scale=None, window=0, **kw):
        err = torch.zeros(1, dtype=torch.int32, device=DEV)
        out = lai.paged_attention(self.q, self.kv, self.batch, scale=scale, window=window, err=err, **kw)
        torch.cuda.synchronize()
        assert int(err) == 0
        o, tol = self.expected(scale, window)
        off = (out.double() - o).abs()
        assert torch.isfinite(out).all()
        worst = float((off / tol).max()) if off.numel() else 0.0
        assert worst <= 1.0, (worst, float(off.max()))
        return out


# ---- writing and reading back -------------------------------------------------------------------
@pytest.mark.parametrize("cache", list(ref.FORMATS))
@pytest.mark.parametrize("dtype", list(ref.DTYPES))
@pytest.mark.parametrize("hd,Hkv,page", [(128, 8, 16), (64, 3, 256), (128, 1, 64)])
def test_append_bits_and_read_back(cache, dtype, hd, Hkv, page):
    # sequences that start in the middle of a page, cross pages, have one token, none, many
    new, keys = [5, 1, 0, 70, 300], [5, 200, 9, 131, 300]
    fmt, dt, g = ref.FORMATS[cache], ref.DTYPES[dtype], gen(hd + page)
    pages, pool = ref.make_pages(keys, page, seed=3)
    kv = lai.PagedKV.allocate(pool, Hkv, page, hd, fmt)
    rows, width = sum(new), Hkv * hd
    # k and v as column blocks of one projection's rows, scales over many powers of two; a row of
    # zeros, one with a single value, the smallest numbers
    x = torch.randn((rows, 3 * width), generator=g, device=DEV) * torch.exp(3 * torch.randn((rows, 1), generator=g, device=DEV))
    x[1, :] = 0
    x[2, width:2 * width] = 0
    x[2, width + 7] = -3.5
    x[3, :] = 1e-42 if dtype == "f32" else 1e-38
    x = x.to(dt)
    k, v = x[:, width:2 * width], x[:, 2 * width:]
    batch = lai.PagedBatch(starts(new), i32(keys), pages.to(DEV))
    before = [t.clone() for t in (kv.k.view(torch.uint8), kv.v.view(torch.uint8))]
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    lai.paged_kv_append(kv, batch, k, v, err=err)
    kr, vr = lai.paged_kv_read(kv, batch, rows, torch.float32, err=err)
    kb, vb = lai.paged_kv_read(kv, batch, rows, torch.bfloat16, err=err)
    assert int(err) == 0
    at = 0
    touched = torch.zeros(kv.k.shape[:3], dtype=torch.bool, device=DEV)
    for s, (n, L) in enumerate(zip(new, keys)):
        p = torch.arange(L - n, L, device=DEV)
        where = pages.to(DEV)[s, p // page].long(), slice(None), p % page
        touched[where] = True
        for rows_, c, sc, r32, r16 in ((k, kv.k, kv.k_scale, kr, kb), (v, kv.v, kv.v_scale, vr, vb)):
            q, scale = ref.stored(rows_[at:at + n].reshape(n, Hkv, hd), fmt)
            got = c.view(torch.int8)[where].view(c.dtype) if cache == "e4m3" else c[where]
            assert torch.equal(ref.codes(got), q)
            if sc is not None:
                assert torch.equal(sc[where].double(), scale[..., 0])
            want = (q * scale).float().flatten(1)  # one F32 product
            assert torch.equal(r32[at:at + n], want)
            assert torch.equal(r16[at:at + n], want.bfloat16())
        at += n
    for t, b in zip((kv.k.view(torch.uint8), kv.v.view(torch.uint8)), before):
        assert torch.equal(t[~touched], b[~touched])  # nothing else was written
    for t in (kv.k_scale, kv.v_scale):
        assert t is None or (t[~touched] == 1).all()


@pytest.mark.parametrize("cache", list(ref.FORMATS))
def test_append_non_finite_rows(cache):
    fmt, hd = ref.FORMATS[cache], 128
    x = torch.randn((4, 2 * hd), generator=gen(1), device=DEV)
    x[0, 3], x[1, hd + 5], x[2, 9] = math.inf, math.nan, -math.inf
    kv = lai.PagedKV.allocate(2, 2, 16, hd, fmt)
    batch = lai.PagedBatch(i32([0, 4]), i32([4]), i32([[1]]))
    lai.paged_kv_append(kv, batch, x, x)
    k, v = lai.paged_kv_read(kv, batch, 4, torch.float32)
    for got in (k.view(4, 2, hd), v.view(4, 2, hd)):
        if cache == "bf16":  # stored as they are
            assert torch.equal(got.nan_to_num(7.0), x.bfloat16().float().view(4, 2, hd).nan_to_num(7.0))
            continue
        bad = torch.zeros((4, 2), dtype=torch.bool)
        bad[0, 0] = bad[1, 1] = bad[2, 0] = True  # the whole row and head, and no other
        assert torch.equal(torch.isnan(got).all(-1).cpu(), bad)
        assert torch.isfinite(got[~bad.to(DEV)]).all()


def test_append_and_read_skip_what_is_wrong():
    hd, page = 64, 16
    kv = lai.PagedKV.allocate(4, 1, page, hd, torch.int8)
    # sequence 0 fine; 1 has a bad page; 2 has more rows than keys; 3 is longer than its table
    new, keys = [2, 2, 3, 1], [2, 20, 1, 33]
    pages = i32([[0, 1], [2, 99], [3, 0], [1, 1]])
    batch = lai.PagedBatch(starts(new), i32(keys), pages)
    x = torch.randn((10, hd), generator=gen(2), device=DEV)  # two rows behind the last sequence
    for err0, part in ((lai.LAI_DEVERR_PAGE | lai.LAI_DEVERR_POSITION, batch),):
        err = torch.zeros(1, dtype=torch.int32, device=DEV)
        lai.paged_kv_append(kv, part, x, x, err=err)
        assert int(err) == err0
        k, v = (torch.full((10, hd), 7.0, device=DEV) for _ in range(2))
        err.zero_()
        lai.paged_kv_read(kv, part, 10, torch.float32, k=k, v=v, err=err)
        assert int(err) == err0
    q, s = ref.stored(x, torch.int8)
    good = [0, 1, 6]  # sequence 0's rows and sequence 2's last, at position 0
    for got in (k, v):
        assert torch.equal(got[good], (q * s).float()[good])
        left = [r for r in range(10) if r not in good]
        assert (got[left] == 7.0).all()


# ---- attention --------------------------------------------------------------------------------
# (new tokens, keys) of each sequence: one token and one key; the edges of 16-key groups, pages
# and key blocks; a long sequence beside short ones; drafted tokens; a prompt from nothing
RAGGED = [([1], [1]), ([1, 1, 1, 1, 1], [1, 16, 17, 128, 129]), ([1, 1, 1], [3000, 5, 777]),
          ([5, 3, 1, 8], [100, 3, 64, 1000]), ([33, 40], [33, 500])]


@pytest.mark.parametrize("new,keys", RAGGED)
@pytest.mark.parametrize("cache", list(ref.FORMATS))
@pytest.mark.parametrize("dtype", list(ref.DTYPES))
def test_attention_ragged(new, keys, cache, dtype):
    Case(new, keys, 16, 8, 128, cache, 16, dtype, seed=len(new)).check()


@pytest.mark.parametrize("H,Hkv,hd,page", [(4, 4, 64, 16), (6, 2, 64, 32), (8, 1, 128, 64),
                                           (5, 1, 128, 128), (16, 1, 64, 256), (16, 16, 64, 16),
                                           (26, 2, 128, 16)])
@pytest.mark.parametrize("cache,dtype", [("bf16", "f32"), ("i8", "f32"), ("e4m3", "bf16")])
def test_attention_heads_and_pages(H, Hkv, hd, page, cache, dtype):
    Case([1, 7, 2], [300, 40, 65], H, Hkv, hd, cache, page, dtype, seed=H).check()


@pytest.mark.parametrize("window", [1, 15, 100, 5000, 2 ** 31 - 1])
@pytest.mark.parametrize("cache,dtype", [("bf16", "bf16"), ("i8", "f32"), ("e4m3", "f32")])
def test_attention_window(window, cache, dtype):
    Case([1, 9, 60, 1], [1000, 300, 60, 4], 8, 4, 64, cache, 32, dtype, seed=window % 97).check(window=window)


# many rows: one tile and its edges, blocks of 128 keys and theirs, several tiles, a long prefix,
# long and short sequences in one batch, a sequence cut over many CTAs. (The kernel for many rows
# needs 8 to 24 rows a sequence and 128 to 256 tiles of 8 rows over all kv heads; "many" below is
# chosen to be above that.)
WIDE = [([64, 65, 63], [64, 200, 129]), ([128], [128]), ([129, 200], [1000, 257]), ([700], [700]),
        ([300, 1, 40], [4000, 777, 40]), ([130], [20000])]


@pytest.mark.parametrize("new,keys", WIDE)
@pytest.mark.parametrize("cache", list(ref.FORMATS))
@pytest.mark.parametrize("dtype", list(ref.DTYPES))
def test_attention_wide(new, keys, cache, dtype):
    Case(new, keys, 16, 8, 128, cache, 32, dtype, seed=len(new) + keys[0]).check()


@pytest.mark.parametrize("H,Hkv,hd,page", [(4, 4, 64, 16), (6, 2, 64, 32), (8, 1, 128, 64),
                                           (3, 1, 128, 128), (16, 1, 64, 256), (2, 2, 128, 16)])
@pytest.mark.parametrize("cache", list(ref.FORMATS))
@pytest.mark.parametrize("dtype", list(ref.DTYPES))
def test_attention_wide_heads_and_pages(H, Hkv, hd, page, cache, dtype):
    Case([850, 300], [1033, 300], H, Hkv, hd, cache, page, dtype, seed=H).check()


@pytest.mark.parametrize("window", [1, 37, 128, 300, 100000])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("cache,dtype", [("bf16", "bf16"), ("i8", "f32"), ("e4m3", "bf16"), ("bf16", "f32")])
def test_attention_wide_window(window, hd, cache, dtype):
    Case([200, 400], [1000, 400], 4, 2, hd, cache, 16, dtype, seed=window % 89).check(window=window)


@pytest.mark.parametrize("cache", list(ref.FORMATS))
@pytest.mark.parametrize("dtype", list(ref.DTYPES))
@pytest.mark.parametrize("hd,Hkv", [(128, 8), (64, 5)])
def test_attention_many_sequences_of_one_token(cache, dtype, hd, Hkv):
    # more work than CTAs: every CTA goes through several items, cut and whole ones
    r = torch.Generator().manual_seed(hd)
    keys = [int(x) for x in torch.randint(1, 3000, (48,), generator=r)]
    Case([1] * 48, keys, 2 * Hkv, Hkv, hd, cache, 64, dtype, seed=5).check()


# ---- rows that see nothing, rows that belong to nobody -------------------------------------------
@pytest.mark.parametrize("cache", list(ref.FORMATS))
@pytest.mark.parametrize("dtype", list(ref.DTYPES))
@pytest.mark.parametrize("many", [1, 60])
def test_attention_rows_without_keys(cache, dtype, many):
    """More rows than keys (the first see nothing), no keys at all, no rows, and rows before the
    first and behind the last sequence."""
    c = Case([3 * many, 0, 4 * many, 2 * many], [3 * many, 50, 4 * many, 2 * many], 4, 2, 64, cache, 16, dtype)
    kv_len = i32([2 * many, 50, 0, 2 * many])
    front, back, n = 5, 7, c.q.shape[0]
    q = torch.cat([c.q[:front] * 0 + 3, c.q, c.q[:back] * 0 + 3])
    out = torch.full_like(q, 9.0)
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    batch = lai.PagedBatch(c.batch.q_start + front, kv_len, c.batch.pages)
    lai.paged_attention(q, c.kv, batch, out=out, err=err)
    assert int(err) == 0
    assert (out[:front] == 9).all() and (out[front + n:] == 9).all()
    got = out[front:front + n].double()
    assert (got[:many] == 0).all()                   # positions -many .. -1
    assert (got[3 * many:7 * many] == 0).all()       # no keys
    c.new, c.keys = [2 * many, 0, 0, 2 * many], [2 * many, 50, 0, 2 * many]
    c.q = torch.cat([c.q[many:3 * many], c.q[7 * many:]])
    o, tol = c.expected()
    got = torch.cat([got[many:3 * many], got[7 * many:]])
    assert ((got - o).abs() <= tol).all()


def test_empty_batches_do_nothing():
    kv = lai.PagedKV.allocate(2, 1, 16, 64, torch.int8)
    none = lai.PagedBatch(i32([0]), i32([]), torch.zeros((0, 1), dtype=torch.int32, device=DEV))
    q = torch.ones((3, 64), device=DEV)
    out = torch.full_like(q, 5.0)
    lai.paged_attention(q, kv, none, out=out)
    lai.paged_kv_append(kv, none, q, q)
    assert (out == 5).all() and not kv.k.any()
    one = lai.PagedBatch(i32([0, 0]), i32([0]), i32([[0]]))
    assert lai.paged_attention(q[:0], kv, one).shape == (0, 64)
    k, v = lai.paged_kv_read(kv, one, 0, torch.float32)
    assert k.shape == v.shape == (0, 64)


# ---- what must not be seen ------------------------------------------------------------------------
@pytest.mark.parametrize("garbage", [math.nan, math.inf, torch.finfo(torch.bfloat16).min])
@pytest.mark.parametrize("new,keys,window", [([1, 1], [37, 300], 0), ([1, 5], [400, 129], 20),
                                             ([150, 70], [350, 70], 0), ([90, 200], [777, 200], 33)])
@pytest.mark.parametrize("cache,dtype", [("bf16", "f32"), ("bf16", "bf16"), ("i8", "f32"), ("e4m3", "bf16")])
def test_attention_garbage_behind_the_keys(garbage, new, keys, window, cache, dtype):
    # pages' ends, spare pages and their scales hold garbage
    Case(new, keys, 16, 8, 128, cache, 64, dtype, seed=9, garbage=garbage).check(window=window)


@pytest.mark.parametrize("new,keys,window", [([6], [50], 0), ([2], [40], 8), ([700], [800], 0), ([600], [900], 60)])
@pytest.mark.parametrize("cache,dtype", [("bf16", "f32"), ("bf16", "bf16"), ("i8", "f32"), ("i8", "bf16"),
                                         ("e4m3", "f32"), ("e4m3", "bf16")])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_attention_non_finite_values_reach_only_who_sees_them(new, keys, window, cache, dtype, bad):
    """A non-finite value in row j of V: tokens before j, and those whose window has passed it, are
    as without it; the others get it (in its column; a whole head's row in an 8-bit cache)."""
    n, L = new[0], keys[0]
    c = Case(new, keys, 4, 2, 128, cache, 16, dtype, seed=3)
    clean = c.check(window=window)
    j, col = L - n + n // 2, 128 + 77  # kv head 1
    row = c.v_rows[j].clone()
    row[col] = bad
    at = lai.PagedBatch(i32([0, 1]), i32([j + 1]), c.batch.pages)
    lai.paged_kv_append(c.kv, at, c.k_rows[j:j + 1], row[None])
    out = lai.paged_attention(c.q, c.kv, c.batch, window=window)
    pos = torch.arange(L - n, L, device=DEV)
    sees = (pos >= j) & (pos < j + (window or L))
    hit = torch.zeros_like(out, dtype=torch.bool).view(n, 4, 128)
    if cache == "bf16":
        hit[sees, 2:, 77] = True
        # An infinity may come out as NaN: a weight w is the sum of its 16-bit terms, the second of
        # either sign (or 0), so w * inf is inf + (-inf) (or 0 * inf) = NaN.
        assert not torch.isfinite(out.view(n, 4, 128)[sees, 2:, 77]).any()
    else:
        hit[sees, 2:] = True
        assert torch.isnan(out.view(n, 4, 128)[sees, 2:]).all()
    hit = hit.view(n, -1)
    assert torch.isfinite(out[~hit]).all()
    if cache == "bf16":  # the rest of these rows too: the row's other values are what they were
        o, tol = c.expected(window=window)
        # (the reference leaves non-finite values out of its sums)
        assert ((out.double() - o).abs() <= tol)[~hit].all()
    else:
        assert torch.equal(out[~sees], clean[~sees])


@pytest.mark.parametrize("n", [4, 1100])
@pytest.mark.parametrize("cache", ["bf16", "i8"])
def test_attention_non_finite_keys_reach_only_who_sees_them(n, cache):
    c = Case([n], [n + 30], 2, 1, 64, cache, 16, "f32", seed=4)
    clean = c.check()
    j = 30 + n // 2
    row = c.k_rows[j].clone()
    row[5] = math.nan
    at = lai.PagedBatch(i32([0, 1]), i32([j + 1]), c.batch.pages)
    lai.paged_kv_append(c.kv, at, row[None], c.v_rows[j:j + 1])
    out = lai.paged_attention(c.q, c.kv, c.batch)
    assert torch.equal(out[:n // 2], clean[:n // 2])
    assert torch.isnan(out[n // 2:]).all()


@pytest.mark.parametrize("n", [2, 400])
def test_attention_bad_pages_and_lengths(n):
    """A page outside the pool counts as not there; a sequence with a length outside its table is
    skipped; the others are computed."""
    L = 2 * n + 100
    c = Case([n, n, n], [L, L, L], 2, 1, 64, "bf16", 16, "f32", seed=6)
    pages = c.batch.pages.clone()
    pages[1, 2] = c.kv.n_pages                      # keys 32..47 of sequence 1
    kv_len = i32([L, L, pages.shape[1] * 16 + 1])
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    out = torch.full_like(c.q, 9.0)
    lai.paged_attention(c.q, c.kv, lai.PagedBatch(c.batch.q_start, kv_len, pages), out=out, err=err)
    assert int(err) == lai.LAI_DEVERR_PAGE | lai.LAI_DEVERR_POSITION
    assert (out[2 * n:] == 9).all()
    kd, vd = ref.codes(c.kv.k), ref.codes(c.kv.v)
    for s in (0, 1):
        k, v = ref.sequence(kd, c.pages[s], L), ref.sequence(vd, c.pages[s], L)
        q = c.q[s * n:(s + 1) * n].double().view(n, 2, 64)
        if s == 1:  # -inf scores for the keys that are gone
            p = torch.arange(L - n, L, device=DEV)[:, None]
            j = torch.arange(L, device=DEV)
            see = (j <= p) & ((j < 32) | (j >= 48))
            w = torch.einsum("nhd,kd->hnk", q, k[:, 0]) / 8
            o = torch.einsum("hnk,kd->nhd", torch.softmax(w.masked_fill(~see, -math.inf), -1), v[:, 0])
        else:
            o = ref.attend(q, k, v, L - n, 0.125)[0]
        assert (out[s * n:(s + 1) * n].double() - o.flatten(1)).abs().max() <= 2e-5
    # q_start that decreases, and a row range outside the rows: flagged, nothing outside is touched
    for q_start in ([0, n, n - 1, 3 * n], [0, n, 2 * n, 3 * n + 1], [-1, n, 2 * n, 3 * n]):
        err.zero_()
        lai.paged_attention(c.q, c.kv, lai.PagedBatch(i32(q_start), i32([L, L, L]), c.batch.pages), out=out, err=err)
        assert int(err) == lai.LAI_DEVERR_POSITION


# ---- numbers --------------------------------------------------------------------------------------
@pytest.mark.parametrize("n", [1, 530])
@pytest.mark.parametrize("cache,dtype", [("bf16", "f32"), ("i8", "f32"), ("e4m3", "bf16"), ("bf16", "bf16")])
@pytest.mark.parametrize("scale", [0.0, -0.1, 1e-6, 3.0])
def test_attention_scales(n, cache, dtype, scale):
    Case([n], [n + 200], 4, 2, 128, cache, 16, dtype, seed=8).check(scale=scale)


@pytest.mark.parametrize("n", [1, 1100])
@pytest.mark.parametrize("dtype", list(ref.DTYPES))
@pytest.mark.parametrize("cache", list(ref.FORMATS))
def test_attention_extreme_scores(n, dtype, cache):
    """All scores far below zero (down to -1e30), rows of equal scores, one key above all others."""
    c = Case([n], [n + 260], 2, 1, 64, cache, 32, dtype, seed=10)
    L = n + 260
    for how in ("low", "equal", "one"):
        k = torch.zeros_like(c.k_rows)
        if how == "low":
            k[:, 0] = -1e30  # the same for every key, so every key weighs the same
        elif how == "one":
            k[7, 0] = 60.0
        lai.paged_kv_append(c.kv, c.whole, k, c.v_rows)
        q = torch.zeros_like(c.q)
        q[:, 0] = 8.0
        q[:, 64] = 8.0
        out = lai.paged_attention(q, c.kv, c.batch, scale=1.0).double().view(n, 2, 64)
        v = ref.sequence(ref.values(c.kv.v, c.kv.v_scale), c.pages[0], L)[:, 0]
        if how == "one":
            want = v[7].expand(n, 64)
        else:
            want = v.cumsum(0)[L - n:] / torch.arange(L - n + 1, L + 1, device=DEV)[:, None]
        tol = 2e-5 if dtype == "f32" else 2.0 ** -6
        assert (out - want[:, None]).abs().max() <= tol


@pytest.mark.parametrize("n", [1, 530])
@pytest.mark.parametrize("cache", ["i8", "e4m3"])
def test_attention_value_scales_over_many_orders(n, cache):
    """Value rows from 2^-40 to 2^40: the weights of small ones must not drown the large ones'."""
    c = Case([n], [n + 300], 2, 1, 64, cache, 16, "f32", seed=11)
    g = gen(5)
    v = c.v_rows * torch.exp2(torch.randint(-40, 41, (c.v_rows.shape[0], 1), generator=g, device=DEV).float())
    lai.paged_kv_append(c.kv, c.whole, c.k_rows, v)
    c.check()


@pytest.mark.parametrize("cache,dtype", [("bf16", "bf16"), ("i8", "f32"), ("bf16", "f32")])
def test_attention_is_deterministic(cache, dtype):
    # long sequences, so that items are cut and joined; the order of arrival must not matter
    c = Case([1, 1, 3], [30000, 9000, 20000], 4, 2, 128, cache, 64, dtype, seed=12)
    scratch = lai.paged_attention_scratch(128)
    first = c.check(scratch=scratch)
    for _ in range(5):
        assert torch.equal(lai.paged_attention(c.q, c.kv, c.batch, scratch=scratch), first)
    c = Case([600], [9000], 4, 2, 128, cache, 64, dtype, seed=13)
    first = c.check(scratch=scratch)  # the same scratch for the other kernel
    for _ in range(5):
        assert torch.equal(lai.paged_attention(c.q, c.kv, c.batch, scratch=scratch), first)
    assert not scratch[:1024].view(torch.int32).any()  # left as it was found


# ---- memory ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("cache", ["i8", "bf16"])
@pytest.mark.parametrize("n", [1, 300])
def test_offsets_beyond_32_bits(cache, n):
    """A pool of more than 2^32 elements, its last pages in use."""
    hd, Hkv, page = 128, 8, 256
    pool = (1 << 32) // (hd * Hkv * page) + 64
    kv = lai.PagedKV.allocate(pool, Hkv, page, hd, ref.FORMATS[cache])
    L = 700
    pages = i32([[pool - 1, pool - 2, pool - 40]])
    g = gen(1)
    k, v = (torch.randn((L, Hkv * hd), generator=g, device=DEV) for _ in range(2))
    lai.paged_kv_append(kv, lai.PagedBatch(i32([0, L]), i32([L]), pages), k, v)
    kr, vr = lai.paged_kv_read(kv, lai.PagedBatch(i32([0, L]), i32([L]), pages), L, torch.float32)
    for x, got in ((k, kr), (v, vr)):
        q, s = ref.stored(x.view(L, Hkv, hd), ref.FORMATS[cache])
        assert torch.equal(got, (q * s).float().flatten(1))
    q = torch.randn((n, Hkv * hd), generator=g, device=DEV)
    out = lai.paged_attention(q, kv, lai.PagedBatch(i32([0, n]), i32([L]), pages))
    o, a, b, u = ref.attend(q.double().view(n, Hkv, hd), kr.double().view(L, Hkv, hd), vr.double().view(L, Hkv, hd), L - n, hd ** -0.5)
    assert ((out.double() - o.flatten(1)).abs() <= ref.tolerance(o, a, b, u, torch.float32, kv.k.dtype).flatten(1)).all()


@pytest.mark.parametrize("n", [1, 530])
def test_strided_rows_other_streams_and_outputs(n):
    H, Hkv, hd = 4, 2, 64
    c = Case([n, n], [n + 100, n], H, Hkv, hd, "e4m3", 16, "f32", seed=14)
    want = c.check()
    wide = torch.full((2 * n, (H + 2 * Hkv) * hd + 12), 7.0, device=DEV)
    wide[:, 4:4 + H * hd] = c.q
    out = torch.empty_like(c.q)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    got = lai.paged_attention(wide[:, 4:4 + H * hd], c.kv, c.batch, out=out, stream=stream)
    stream.synchronize()
    assert got is out and torch.equal(out, want)
    with torch.cuda.stream(stream):  # the current stream is the default
        x = wide[:, 4:4 + Hkv * hd]
        lai.paged_kv_append(c.kv, c.batch, x, x)
        buf = torch.full((2 * n, 3 * Hkv * hd), 5.0, device=DEV)
        lai.paged_kv_read(c.kv, c.batch, 2 * n, torch.float32, k=buf[:, :Hkv * hd], v=buf[:, 2 * Hkv * hd:])
    stream.synchronize()
    q, s = ref.stored(x.reshape(2 * n, Hkv, hd), torch.float8_e4m3fn)
    assert torch.equal(buf[:, :Hkv * hd], (q * s).float().flatten(1))
    assert torch.equal(buf[:, 2 * Hkv * hd:], buf[:, :Hkv * hd])
    assert (buf[:, Hkv * hd:2 * Hkv * hd] == 5).all()


@pytest.mark.parametrize("n", [1, 200])
@pytest.mark.parametrize("cache", ["bf16", "i8"])
def test_captured_in_a_graph_and_replayed_with_other_lengths(n, cache):
    """Append and attention as one graph; rows, lengths and pages change between replays."""
    H, Hkv, hd, page, S = 4, 2, 64, 16, 3
    big = Case([n] * S, [600 + n] * S, H, Hkv, hd, cache, page, "f32", seed=15)
    kv, scratch = big.kv, lai.paged_attention_scratch(hd)
    rows = torch.zeros((S * n, (H + 2 * Hkv) * hd), device=DEV)
    kv_len, pages = big.batch.kv_len, big.batch.pages
    q, k, v = rows[:, :H * hd], rows[:, H * hd:(H + Hkv) * hd], rows[:, (H + Hkv) * hd:]
    out = torch.empty((S * n, H * hd), device=DEV)
    err = torch.zeros(1, dtype=torch.int32, device=DEV)

    def step():
        lai.paged_kv_append(kv, big.batch, k, v, err=err)
        lai.paged_attention(q, kv, big.batch, scratch=scratch, out=out, err=err)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for seed, lens in enumerate(([n, n + 1, n + 599], [n + 300, n, n + 17], [n + 64, n + 128, n + 256])):
        rows.copy_(torch.randn(rows.shape, generator=gen(seed), device=DEV))
        kv_len.copy_(i32(lens))
        pages.copy_(pages[torch.randperm(S)])
        graph.replay()
        torch.cuda.synchronize()
        assert int(err) == 0
        kd, vd = ref.values(kv.k, kv.k_scale), ref.values(kv.v, kv.v_scale)
        for s, L in enumerate(lens):
            o, a, b, u = ref.attend(q[s * n:(s + 1) * n].double().reshape(n, H, hd), ref.sequence(kd, pages[s], L),
                                 ref.sequence(vd, pages[s], L), L - n, hd ** -0.5)
            tol = ref.tolerance(o, a, b, u, torch.float32, kv.k.dtype).flatten(1)
            assert ((out[s * n:(s + 1) * n].double() - o.flatten(1)).abs() <= tol).all()


def test_calls_at_once_with_a_scratch_each():
    cases = [Case([1, 1], [5000, 900], 8, 4, 128, "i8", 64, "f32", seed=20),
             Case([200], [2000], 8, 4, 128, "bf16", 64, "bf16", seed=21)]
    want = [c.check() for c in cases]
    streams = [torch.cuda.Stream() for _ in range(4)]
    scratch = [lai.paged_attention_scratch(128) for _ in streams]
    torch.cuda.synchronize()
    outs = []
    for i in range(40):
        s = i % 4
        outs.append((i % 2, lai.paged_attention(cases[i % 2].q, cases[i % 2].kv, cases[i % 2].batch,
                                                scratch=scratch[s], out=torch.empty_like(want[i % 2]), stream=streams[s])))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[k]) for k, o in outs)


# ---- together -------------------------------------------------------------------------------------
@pytest.mark.parametrize("cache", list(ref.FORMATS))
@pytest.mark.parametrize("dtype", list(ref.DTYPES))
def test_prompt_then_tokens_equals_attention_over_the_whole_sequence(cache, dtype):
    """What a server does: prompts in chunks, then tokens, with pages given out as they are
    needed. Every output equals attention over all rows so far."""
    H, Hkv, hd, page, S = 4, 2, 128, 16, 2
    dt, g = ref.DTYPES[dtype], gen(16)
    kv = lai.PagedKV.allocate(128, Hkv, page, hd, ref.FORMATS[cache])
    free = torch.randperm(128, generator=torch.Generator().manual_seed(1)).tolist()
    pages = torch.full((S, 64), -1, dtype=torch.int32)
    scratch, err = lai.paged_attention_scratch(hd), torch.zeros(1, dtype=torch.int32, device=DEV)
    lens, kept = [0] * S, [[] for _ in range(S)]
    for new in ([600, 237], [90, 1], [1, 70], [1, 1], [1, 1], [5, 1]):
        for s, n in enumerate(new):
            lens[s] += n
            for j in range(-(-lens[s] // page)):
                if pages[s, j] < 0:
                    pages[s, j] = free.pop()
        rows = sum(new)
        x = torch.randn((rows, (H + 2 * Hkv) * hd), generator=g, device=DEV).to(dt)
        q, k, v = x[:, :H * hd], x[:, H * hd:(H + Hkv) * hd], x[:, (H + Hkv) * hd:]
        batch = lai.PagedBatch(starts(new), i32(lens), pages.to(DEV))
        lai.paged_kv_append(kv, batch, k, v, err=err)
        out = lai.paged_attention(q, kv, batch, scratch=scratch, err=err)
        at = 0
        for s, n in enumerate(new):
            kept[s].append((k[at:at + n].reshape(n, Hkv, hd), v[at:at + n].reshape(n, Hkv, hd)))
            ks, vs = (torch.cat([torch.mul(*ref.stored(r[i], kv.k.dtype)) for r in kept[s]]) for i in (0, 1))
            o, a, b, u = ref.attend(q[at:at + n].double().reshape(n, H, hd), ks, vs, lens[s] - n, hd ** -0.5)
            tol = ref.tolerance(o, a, b, u, dt, kv.k.dtype).flatten(1)
            assert ((out[at:at + n].double() - o.flatten(1)).abs() <= tol).all()
            at += n
    assert int(err) == 0


def test_same_as_decode_attention_over_its_dense_cache():
    """One token per sequence over BF16 values: the paged kernel and lai.decode_attention on the
    same keys."""
    S, H, Hkv, hd, L = 3, 16, 8, 128, [1, 300, 999]
    c = Case([1] * S, L, H, Hkv, hd, "bf16", 64, "f32", seed=17)
    kc, vc = (torch.zeros((S, 1000, Hkv * hd), device=DEV) for _ in range(2))
    k, v = lai.paged_kv_read(c.kv, c.whole, sum(L), torch.float32)
    at = 0
    for s, n in enumerate(L):
        kc[s, :n], vc[s, :n] = k[at:at + n], v[at:at + n]
        at += n
    last = torch.tensor([sum(L[:s + 1]) - 1 for s in range(S)], device=DEV)
    dense = lai.decode_attention(c.q, k[last].contiguous(), v[last].contiguous(), kc, vc, i32([n - 1 for n in L]), H, Hkv)
    assert (dense - c.check()).abs().max() <= 1e-5


# ---- anything -------------------------------------------------------------------------------------
@pytest.mark.parametrize("seed", range(40))
def test_attention_random(seed):
    import random
    r = random.Random(seed)
    hd, Hkv = r.choice([64, 128]), r.choice([1, 2, 3, 5, 8])
    H = Hkv * r.randint(1, 16 if Hkv < 3 else 4)
    S = r.randint(1, 12)
    top = r.choice([3, 40, 300])
    new = [r.randint(0, top) for _ in range(S)]
    keys = [n + (r.randint(0, r.choice([1, 200, 1500])) if r.random() < 0.8 else 0) for n in new]
    c = Case(new, keys, H, Hkv, hd, r.choice(list(ref.FORMATS)), r.choice([16, 32, 64, 128, 256]),
             r.choice(list(ref.DTYPES)), seed=seed, garbage=math.nan)
    c.check(window=r.choice([0, 0, r.randint(1, 400)]))


@pytest.mark.parametrize("top", [1, 40])
@pytest.mark.parametrize("cache,dtype", [("i8", "f32"), ("bf16", "bf16")])
def test_more_sequences_than_are_kept_at_hand(top, cache, dtype):
    """700 sequences: the schedule's table of sequences in shared memory holds 256."""
    import random
    r = random.Random(top)
    new = [r.randint(0 if top > 1 else 1, top) for _ in range(700)]
    keys = [n + r.choice([0, 3, r.randint(0, 300)]) for n in new]
    Case(new, keys, 4, 2, 64, cache, 16, dtype, seed=23).check()


@pytest.mark.parametrize("n", [6, 1100])
@pytest.mark.parametrize("cache,dtype", [("i8", "f32"), ("bf16", "bf16"), ("bf16", "f32"), ("e4m3", "bf16")])
def test_attention_non_finite_queries_stay_in_their_rows(n, cache, dtype):
    c = Case([n], [n + 40], 2, 1, 64, cache, 16, dtype, seed=24)
    clean = c.check()
    q = c.q.clone()
    q[n // 2, 70] = math.nan      # head 1 of one token
    q[n // 3, 5] = math.inf       # head 0 of another
    out = lai.paged_attention(q, c.kv, c.batch).view(n, 2, 64)
    hit = torch.zeros((n, 2), dtype=torch.bool, device=DEV)
    hit[n // 2, 1] = hit[n // 3, 0] = True
    assert torch.isnan(out[hit]).all()
    # The other rows keep the bounds of every row, not their bits: whether a block's weights come
    # from the polynomial or the hardware's exponential is voted by the 32 rows of a warp (scores of
    # 2^20 and more, and infinities, need the second), and either is within the bound of a row.
    o, tol = (t.view(n, 2, 64)[~hit] for t in c.expected())
    assert ((out[~hit].double() - o).abs() <= tol).all()
    assert ((clean.view(n, 2, 64)[~hit].double() - o).abs() <= tol).all()


@pytest.mark.parametrize("cache,dtype", [("bf16", "f32"), ("bf16", "bf16"), ("i8", "f32"), ("e4m3", "bf16")])
@pytest.mark.parametrize("S,new,H,Hkv", [(48, 1, 16, 8), (200, 1, 16, 8), (6, 90, 16, 8)])
def test_attention_same_bits_in_every_call(S, new, H, Hkv, cache, dtype):
    """Rings of copies and joined parts: 200 calls in a row give the first one's bits."""
    import random
    r = random.Random(S)
    keys = [new + r.randint(0, 3000 if S < 100 else 700) for _ in range(S)]
    c = Case([new] * S, keys, H, Hkv, 128, cache, 64 if S < 100 else 16, dtype, seed=S)
    first = c.check()
    scratch = lai.paged_attention_scratch(128)
    outs = [torch.empty_like(first) for _ in range(50)]
    for _ in range(4):
        for o in outs:
            lai.paged_attention(c.q, c.kv, c.batch, scratch=scratch, out=o)
        assert all(torch.equal(o, first) for o in outs)


@pytest.mark.parametrize("n", [1, 150])
@pytest.mark.parametrize("cache,dtype", [("bf16", "bf16"), ("i8", "f32"), ("e4m3", "bf16"), ("bf16", "f32")])
def test_attention_over_shared_pages(n, cache, dtype):
    """A common prefix held once for three sequences, and a page that one table names twice."""
    c = Case([n] * 3, [n + 260] * 3, 16, 8, 128, cache, 32, dtype, seed=25)
    c.pages[1:, :8] = c.pages[0, :8]
    c.pages[2, 5] = c.pages[2, 4]
    c.batch = lai.PagedBatch(c.batch.q_start, c.batch.kv_len, c.pages.to(DEV))
    c.check()


@pytest.mark.parametrize("cache", list(ref.FORMATS))
def test_append_attend_and_read_on_one_stream_many_steps(cache):
    """A decode loop without a synchronisation: every step sees the keys that the ones before wrote."""
    S, H, Hkv, hd, page, steps = 5, 8, 4, 64, 16, 40
    g = gen(26)
    pages, pool = ref.make_pages([steps + 7 * s for s in range(S)], page, seed=26)
    kv = lai.PagedKV.allocate(pool, Hkv, page, hd, ref.FORMATS[cache])
    kv_len = i32([7 * s for s in range(S)])
    batch = lai.PagedBatch(starts([1] * S), kv_len, pages.to(DEV))
    # the keys that are there already
    old = [7 * s for s in range(S)]
    x = torch.randn((2, sum(old), Hkv * hd), generator=g, device=DEV)
    lai.paged_kv_append(kv, lai.PagedBatch(starts(old), i32(old), pages.to(DEV)), x[0], x[1])
    rows = torch.randn((steps, S, (H + 2 * Hkv) * hd), generator=g, device=DEV)
    scratch = lai.paged_attention_scratch(hd)
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    outs = []
    for t in range(steps):
        kv_len.add_(1)
        q, k, v = rows[t].split([H * hd, Hkv * hd, Hkv * hd], dim=1)
        lai.paged_kv_append(kv, batch, k, v, err=err)
        outs.append(lai.paged_attention(q, kv, batch, scratch=scratch, err=err))
    assert int(err) == 0
    kd, vd = ref.values(kv.k, kv.k_scale), ref.values(kv.v, kv.v_scale)
    for s in range(S):
        keys = ref.sequence(kd, pages[s], old[s] + steps), ref.sequence(vd, pages[s], old[s] + steps)
        for t in (0, 1, 17, steps - 1):
            n = old[s] + t + 1
            q = rows[t, s, :H * hd].double().view(1, H, hd)
            o, a, b, u = ref.attend(q, keys[0][:n], keys[1][:n], n - 1, hd ** -0.5, 0)
            tol = ref.tolerance(o, a, b, u, torch.float32, ref.FORMATS[cache]).flatten()
            assert ((outs[t][s].double() - o.flatten()).abs() <= tol).all()
