"""The TTS decode frame over a paged cache: the oracle's frame (test_gpu_tts_frame.py) with keys and
values as the cache's format holds them.

Tolerance: a key or value within the GPU's and the oracle's rounding difference (about 1e-6) of a
boundary between two stored values may fall to either side. With some 10^4 values stored and steps
of 2^-8 to 2^-4 of a value that happens a few times in a test. One such step, at most 1/16 of a value
near 1 in one of 2048 attention outputs, moves a residual element by 1/16 * 2048^-1/2 = 1.4e-3 and a
logit by about as much; 5e-3 leaves room for a few, where wrong wiring gives errors near 1.
"""
import dataclasses

import numpy as np
import pytest

import lai
import paged_ref as ref
import runner
import test_gpu_tts_frame as base
from conftest import max_rel_err

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
TOL = 5e-3


class StoredOracleFrame(base.OracleFrame):
    def __init__(self, tf):
        super().__init__(tf)
        self.kept = {"kc": self.kc, "vc": self.vc}
        self.fmt = ref.FORMATS[tf.cfg.kv_cache]

    def layers(self, x, layers, kc, vc, pos, inter):
        if kc is not self.kc:  # the code predictor's cache is dense F32
            return super().layers(x, layers, kc, vc, pos, inter)
        oracle, c, hd = base.oracle, self.c, self.c.head_dim
        qd, kvd = c.n_q * hd, c.n_kv * hd

        def stored(row):
            q, s = ref.stored(torch.from_numpy(np.ascontiguousarray(row)).view(c.n_kv, hd), self.fmt)
            return (q * s).float().reshape(-1).numpy()

        for i, L in enumerate(layers):
            qkv = oracle.linear_bf16(oracle.rms_norm(x, L["in_norm"], c.eps), L["wqkv"])
            q, k = oracle.qk_norm_rope(qkv[:, :qd], qkv[:, qd:qd + kvd], L["q_norm"], L["k_norm"], self.cos,
                                       self.sin, np.array([pos], np.int32), c.n_q, c.n_kv, hd, c.eps, bf16=False)
            kc[i, 0, pos], vc[i, 0, pos] = stored(k[0]), stored(qkv[0, qd + kvd:])
            attn = oracle.decode_attention(q, kc[i], vc[i], np.array([pos], np.int32), c.n_q, c.n_kv, hd)
            x = oracle.add_inplace(x, oracle.linear_bf16(attn, L["wo"]))
            gu = oracle.linear_bf16(oracle.rms_norm(x, L["post_norm"], c.eps), L["wgu"])
            x = oracle.add_inplace(x, oracle.linear_bf16(oracle.swiglu_multiply(gu, inter), L["wd"]))
        return x


@pytest.mark.parametrize("kv_cache", list(ref.FORMATS))
def test_frames_over_a_paged_cache_match_the_oracle(kv_cache, monkeypatch):
    frames, cfg = 3, dataclasses.replace(base.CFG, kv_cache=kv_cache, kv_page=16)
    tf = runner.TtsFrame(cfg, frames, seed=5)
    ora = StoredOracleFrame(tf)
    monkeypatch.setattr(base, "TOL", TOL)
    tf.record = []
    for _ in range(frames):
        tf.frame()
    torch.cuda.synchronize()
    assert int(tf.err.item()) == 0 and int(tf.kv_len.item()) == frames + 1
    recorded = [base.np32(r) for r in tf.record]
    for f in range(frames):
        ora.frame(f, tf.codes.cpu().numpy(), recorded)


@pytest.mark.parametrize("kv_cache", list(ref.FORMATS))
def test_paged_frames_as_a_graph_equal_direct_launches(kv_cache):
    frames, cfg = 3, dataclasses.replace(base.CFG, kv_cache=kv_cache, kv_page=16)
    a, b = runner.TtsFrame(cfg, frames, seed=9), runner.TtsFrame(cfg, frames, seed=9)
    for _ in range(frames):
        a.frame()
        b.frame(graph=True)
    torch.cuda.synchronize()
    assert torch.equal(a.codes, b.codes) and torch.equal(a.codec_sum, b.codec_sum)
    for x, y in zip(a.kc, b.kc):
        assert torch.equal(x.k.view(torch.uint8), y.k.view(torch.uint8))
    # what the cache stands for is what the dense frame keeps, up to the format's half step (the
    # first frame's keys come from the same input in both)
    c = runner.TtsFrame(base.CFG, frames, seed=9)
    c.frame()
    k, _ = lai.paged_kv_read(a.kc[0], lai.PagedBatch(torch.tensor([0, 1], dtype=torch.int32, device="cuda"),
                                                     torch.ones(1, dtype=torch.int32, device="cuda"), a.batch.pages),
                             1, torch.float32)
    half = {"bf16": 2.0 ** -8, "e4m3": 2.0 ** -4, "i8": 0.5 / 127}[kv_cache]
    want = c.kc[0][0, :1]
    off = (k - want).abs().view(8, 128)
    size = want.abs().view(8, 128) if kv_cache == "bf16" else want.abs().view(8, 128).amax(-1, keepdim=True)
    assert (off <= size * half * 1.01 + 1e-5).all()
    assert max_rel_err(k.cpu().numpy(), want.cpu().numpy()) < 1
