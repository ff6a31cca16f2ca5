"""What the paged cache's binding makes and checks by itself, on the host: no kernel runs."""
import contextlib
import types

import pytest

import lai

torch = pytest.importorskip("torch")


@pytest.fixture
def calls(monkeypatch):
    """CPU tensors in place of CUDA ones; the entry points only note their arguments. .made: every
    tensor that the binding makes, and the stream that was current then; .recorded: tensors that
    were told of another stream."""
    got = types.SimpleNamespace(made=[], recorded=[], entries=[], current="theirs")

    @contextlib.contextmanager
    def stream(s):
        was, got.current = got.current, s
        yield
        got.current = was

    def note(fn):
        def made(*a, **kw):
            t = fn(*a, **{k: v for k, v in kw.items() if k != "device"})
            got.made.append((t.data_ptr(), got.current))
            return t
        return made

    monkeypatch.setattr(torch.cuda, "stream", stream)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *a: got.current)
    monkeypatch.setattr(lai, "_need_cuda", lambda *a: None)
    monkeypatch.setattr(lai, "_paged_call", lambda fn, index, s, *a: got.entries.append((fn.__name__, s, a)))
    for name in ("empty", "zeros", "empty_like", "empty_strided"):
        monkeypatch.setattr(torch, name, note(getattr(torch, name)))
    monkeypatch.setattr(torch.Tensor, "new_empty", note(torch.Tensor.new_empty))
    monkeypatch.setattr(torch.Tensor, "record_stream", lambda t, s: got.recorded.append((t.data_ptr(), s)), raising=False)
    return got


def cache(dtype=torch.bfloat16):
    return lai.PagedKV(torch.ones((4, 2, 16, 64), dtype=dtype), torch.ones((4, 2, 16, 64), dtype=dtype))


def batch(*q_start):
    n = len(q_start) - 1
    return lai.PagedBatch(torch.tensor(q_start, dtype=torch.int32), torch.ones(n, dtype=torch.int32),
                          torch.tensor([[0, 1]] * n, dtype=torch.int32))


@pytest.mark.parametrize("given", [False, True])
def test_what_a_call_makes_is_made_in_its_streams_order(calls, given):
    """Scratch that is zeroed, or memory that is given back, in another stream's order than the
    kernel's would be written under it."""
    kv, b, q = cache(), batch(0, 3), torch.ones((3, 256))
    mine = types.SimpleNamespace(cuda_stream=7) if given else None
    calls.made.clear()
    out = lai.paged_attention(q, kv, b, stream=mine)
    k, v = lai.paged_kv_read(kv, b, 3, torch.float32, stream=mine)
    want = mine if given else "theirs"
    assert len(calls.made) >= 4 and all(s is want for _, s in calls.made)
    assert [s for _, s, _ in calls.entries] == [mine, mine]
    # what the caller gets is also known to the stream that they will use it on
    assert calls.recorded == ([(t.data_ptr(), "theirs") for t in (out, k, v)] if given else [])


def test_scratch_is_zeroed_where_the_kernels_count():
    a = lai.paged_attention_scratch(64, "cpu")
    assert a.nbytes == lai.load().lai_paged_attention_scratch_bytes(64)
    assert not a[:1024].view(torch.int32).any()


@pytest.mark.parametrize("given", [False, True])
def test_decode_attention_makes_its_own_in_its_streams_order(calls, given, monkeypatch):
    mine = types.SimpleNamespace(cuda_stream=7) if given else None
    monkeypatch.setattr(lai, "call", lambda *a: calls.entries.append(a))
    monkeypatch.setattr(lai, "_s", lambda s: s)
    kc, vc = torch.ones((2, 32, 256)), torch.ones((2, 32, 256))
    row = torch.ones((2, 256))
    calls.made.clear()
    out = lai.decode_attention(torch.ones((2, 512)), row, row, kc, vc, torch.ones(2, dtype=torch.int32), 4, 2, stream=mine)
    assert len(calls.made) == 2 and all(s is (mine if given else "theirs") for _, s in calls.made)
    assert calls.recorded == ([(out.data_ptr(), "theirs")] if given else [])


def test_a_single_row_needs_no_stride(calls):
    """One token's k and v as column blocks of different tensors, at any stride."""
    kv, b = cache(), batch(0, 1)
    k, v = torch.ones((1, 301))[:, 8:136], torch.ones((1, 128))
    lai.paged_kv_append(kv, b, k, v)
    lai.paged_attention(torch.ones((1, 999))[:, :256], kv, b, out=torch.ones((1, 256)))
    assert [a[4] for name, _, a in calls.entries if "append" in name] == [128]
    assert [a[2] for name, _, a in calls.entries if "attention" in name] == [256]


def test_read_makes_one_of_k_and_v_beside_the_other(calls):
    kv, b, buf = cache(), batch(0, 3), torch.ones((3, 400))
    for kw in (dict(k=buf[:, 16:144]), dict(v=buf[:, 16:144])):
        k, v = lai.paged_kv_read(kv, b, 3, torch.float32, **kw)
        assert k.shape == v.shape == (3, 128) and k.stride() == v.stride() == (400, 1)
        assert calls.entries[-1][2][2] == 400


def test_windows_of_any_length(calls):
    kv, b, q = cache(), batch(0, 3), torch.ones((3, 256))
    for window, want in ((0, 0), (7, 7), (2 ** 31 - 1, 2 ** 31 - 1), (2 ** 31, 2 ** 31 - 1), (2 ** 32 + 5, 2 ** 31 - 1)):
        lai.paged_attention(q, kv, b, window=window)
        assert calls.entries[-1][2][8] == want
    for window in (-1, -2 ** 32):
        with pytest.raises(ValueError):
            lai.paged_attention(q, kv, b, window=window)


def test_refuses_a_scratch_that_only_looks_large(calls):
    kv, b, q = cache(), batch(0, 3), torch.ones((3, 256))
    with pytest.raises(ValueError):
        lai.paged_attention(q, kv, b, scratch=torch.ones(1).expand(lai._paged_scratch_floats(64)))
