"""What the paged cache's entry points and their binding refuse, on the host. No kernel runs: each
call returns from a check (or has nothing to do)."""
import ctypes

import pytest

import lai
from conftest import arena_ptr

torch = pytest.importorskip("torch")
MB = 1 << 20


def P(off):
    return arena_ptr(off).value


def kv(**kw):
    f = dict(k=P(0), v=P(4 * MB), k_scale=None, v_scale=None, n_pages=4, page_size=16, n_kv_heads=2,
             head_dim=64, format=lai.LAI_KV_BF16)
    f.update(kw)
    return lai._PagedKVC(*(f[n] for n, _ in lai._PagedKVC._fields_))


def kv8(**kw):
    return kv(**{**dict(format=lai.LAI_KV_I8, k_scale=P(8 * MB), v_scale=P(9 * MB)), **kw})


def batch(**kw):
    f = dict(q_start=P(12 * MB), kv_len=P(13 * MB), pages=P(14 * MB), n_seqs=2, max_pages=8)
    f.update(kw)
    return lai._PagedBatchC(*(f[n] for n, _ in lai._PagedBatchC._fields_))


def append(c, b, k=P(16 * MB), v=P(17 * MB), ld=128, rows=4, dtype="f32"):
    return getattr(lai.load(), f"lai_paged_kv_append_{dtype}")(
        c and ctypes.byref(c), b and ctypes.byref(b), k, v, ld, rows, None, None)


def read(c, b, k=P(16 * MB), v=P(17 * MB), ld=128, rows=4, dtype="f32"):
    return getattr(lai.load(), f"lai_paged_kv_read_{dtype}")(
        k, v, ld, rows, c and ctypes.byref(c), b and ctypes.byref(b), None, None)


def attend(c, b, out=P(16 * MB), q=P(17 * MB), ld=256, rows=4, heads=4, window=0, scratch=P(20 * MB), dtype="f32"):
    return getattr(lai.load(), f"lai_paged_attention_{dtype}")(
        out, q, ld, rows, heads, c and ctypes.byref(c), b and ctypes.byref(b), 0.1, window, scratch, None, None)


BAD_KV = [dict(k=None), dict(v=None), dict(n_pages=0), dict(page_size=0), dict(page_size=24), dict(page_size=512),
          dict(page_size=8), dict(n_kv_heads=0), dict(head_dim=96), dict(head_dim=256), dict(format=3),
          dict(format=-1), dict(format=lai.LAI_KV_I8), dict(format=lai.LAI_KV_E4M3, k_scale=P(8 * MB)),
          dict(k_scale=P(8 * MB), v_scale=P(9 * MB)), dict(k=P(4)), dict(v=P(4 * MB + 8))]
BAD_BATCH = [dict(q_start=None), dict(kv_len=None), dict(pages=None), dict(n_seqs=-1), dict(max_pages=0)]


@pytest.mark.parametrize("call", [append, read, attend])
def test_refuses_malformed_caches_and_batches(call):
    for bad in BAD_KV:
        assert call(kv(**bad), batch()) == lai.LAI_ERR_INVALID, bad
    assert call(kv8(k_scale=P(8 * MB + 4)), batch()) == lai.LAI_ERR_INVALID
    for bad in BAD_BATCH:
        assert call(kv(), batch(**bad)) == lai.LAI_ERR_INVALID, bad
    assert call(None, batch()) == lai.LAI_ERR_INVALID
    assert call(kv(), None) == lai.LAI_ERR_INVALID
    assert call(kv(), batch(), rows=-1) == lai.LAI_ERR_INVALID
    assert call(kv(n_pages=1 << 31), batch()) == lai.LAI_ERR_RANGE
    assert call(kv(), batch(), rows=1 << 31) == lai.LAI_ERR_RANGE
    assert call(kv(), batch(max_pages=1 << 27)) == lai.LAI_ERR_RANGE
    assert call(kv(), batch(), rows=0) == lai.LAI_OK
    assert call(kv(), batch(n_seqs=0)) == lai.LAI_OK


@pytest.mark.parametrize("call", [append, read])
def test_refuses_rows(call):
    c, b = kv(), batch()
    assert call(c, b, k=None) == lai.LAI_ERR_INVALID
    assert call(c, b, v=None) == lai.LAI_ERR_INVALID
    assert call(c, b, ld=124) == lai.LAI_ERR_INVALID             # shorter than a row
    assert call(c, b, ld=130) == lai.LAI_ERR_INVALID             # rows not 16-byte aligned
    assert call(c, b, ld=132, dtype="bf16") == lai.LAI_ERR_INVALID
    assert call(c, b, k=P(16 * MB + 4)) == lai.LAI_ERR_INVALID
    assert call(c, b, k=P(0)) == lai.LAI_ERR_ALIAS               # rows in the cache
    assert call(kv8(), b, v=P(9 * MB)) == lai.LAI_ERR_ALIAS      # rows in the scales
    if call is append:
        assert call(kv(v=P(0)), b) == lai.LAI_ERR_ALIAS          # k and v in one place
        assert call(kv8(v_scale=P(8 * MB)), b) == lai.LAI_ERR_ALIAS
    else:
        assert call(c, b, k=P(16 * MB), v=P(16 * MB)) == lai.LAI_ERR_ALIAS
        assert call(c, b, k=P(16 * MB), v=P(16 * MB + 256), ld=256) == lai.LAI_ERR_ALIAS  # columns overlap


def test_attention_refuses():
    c, b = kv(), batch()
    assert attend(c, b, out=None) == lai.LAI_ERR_INVALID
    assert attend(c, b, q=None) == lai.LAI_ERR_INVALID
    assert attend(c, b, scratch=None) == lai.LAI_ERR_INVALID
    assert attend(c, b, heads=0) == lai.LAI_ERR_INVALID
    assert attend(c, b, heads=3) == lai.LAI_ERR_INVALID          # not a multiple of the kv heads
    assert attend(c, b, heads=34, ld=34 * 64) == lai.LAI_ERR_INVALID  # a group of 17
    assert attend(c, b, window=-1) == lai.LAI_ERR_INVALID
    assert attend(c, b, ld=252) == lai.LAI_ERR_INVALID
    assert attend(c, b, ld=258) == lai.LAI_ERR_INVALID
    assert attend(c, b, q=P(17 * MB + 8)) == lai.LAI_ERR_INVALID
    assert attend(c, b, out=P(16 * MB + 8)) == lai.LAI_ERR_INVALID
    assert attend(c, b, scratch=P(20 * MB + 4)) == lai.LAI_ERR_INVALID
    assert attend(c, b, out=P(17 * MB)) == lai.LAI_ERR_ALIAS     # out on q
    assert attend(c, b, out=P(4 * MB)) == lai.LAI_ERR_ALIAS      # out in the cache
    assert attend(c, b, scratch=P(16 * MB)) == lai.LAI_ERR_ALIAS
    assert attend(c, b, scratch=P(0)) == lai.LAI_ERR_ALIAS
    assert attend(c, b, rows=1 << 28) == lai.LAI_ERR_RANGE
    assert attend(kv(n_kv_heads=64, n_pages=1), batch(n_seqs=1 << 20, max_pages=1 << 20), heads=64, ld=64 * 64) in (
        lai.LAI_ERR_RANGE, lai.LAI_ERR_ALIAS)
    L = lai.load()
    assert L.lai_paged_attention_scratch_bytes(64) > 0 and L.lai_paged_attention_scratch_bytes(128) > 0
    assert L.lai_paged_attention_scratch_bytes(96) == 0


def test_binding_refuses():
    z = torch.zeros
    k8, s8 = z(4, 2, 16, 64, dtype=torch.int8), z(4, 2, 16)
    kb = z(4, 2, 16, 64, dtype=torch.bfloat16)
    for a in [(kb.float(), kb.float()), (kb, k8), (kb.half(), kb.half())]:
        with pytest.raises(TypeError):
            lai.PagedKV(*a)
    for a in [(k8, k8), (k8, k8, s8), (kb, kb, s8, s8), (kb[:2], kb), (kb[0], kb[0]), (kb.transpose(0, 1),) * 2,
              (k8, k8, s8.double(), s8), (k8, k8, s8[:2], s8[:2]), (kb[:, :, :15].contiguous(),) * 2,
              (kb[..., :32].contiguous(),) * 2,
              (kb, kb.clone())]:  # the last: CPU tensors
        with pytest.raises(ValueError):
            lai.PagedKV(*a)
    i = lambda *s: z(*s, dtype=torch.int32)  # noqa: E731
    for a in [(i(3).long(), i(2), i(2, 4)), (i(2), i(2), i(2, 4)), (i(3), i(2), i(3, 4)), (i(3), i(2), i(4)),
              (i(3), i(2), i(4, 2).T), (i(3), i(2), i(2, 4))]:
        with pytest.raises(ValueError):
            lai.PagedBatch(*a)
    with pytest.raises(TypeError):
        lai._paged_fn("lai_paged_attention", torch.float16)
    with pytest.raises(ValueError):
        lai._paged_rows(z(3, 8, 2)[..., 0], 8)
    with pytest.raises(ValueError):
        lai._need_cuda(0, z(3))
