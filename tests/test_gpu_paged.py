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
            o, a, b = ref.attend(q, ref.sequence(kd, self.pages[s], L),
                                 ref.sequence(vd, self.pages[s], L), L - n, scale, window)
            os.append(o.flatten(1))
            tols.append(ref.tolerance(o, a, b, self.dtype, self.cache).flatten(1))
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
# long and short sequences in one batch, a sequence cut over many CTAs
WIDE = [([64, 65, 63], [64, 200, 129]), ([128], [128]), ([129, 200], [1000, 257]), ([700], [700]),
        ([300, 1, 40], [4000, 777, 40]), ([100], [20000])]


@pytest.mark.parametrize("new,keys", WIDE)
@pytest.mark.parametrize("cache", list(ref.FORMATS))
@pytest.mark.parametrize("dtype", list(ref.DTYPES))
def test_attention_wide(new, keys, cache, dtype):
    Case(new, keys, 8, 4, 128, cache, 32, dtype, seed=len(new) + keys[0]).check()


@pytest.mark.parametrize("H,Hkv,hd,page", [(4, 4, 64, 16), (6, 2, 64, 32), (8, 1, 128, 64),
                                           (3, 1, 128, 128), (16, 1, 64, 256), (2, 2, 128, 16)])
@pytest.mark.parametrize("cache", list(ref.FORMATS))
@pytest.mark.parametrize("dtype", list(ref.DTYPES))
def test_attention_wide_heads_and_pages(H, Hkv, hd, page, cache, dtype):
    Case([150, 90], [333, 90], H, Hkv, hd, cache, page, dtype, seed=H).check()


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
