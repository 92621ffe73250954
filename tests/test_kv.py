"""What the paged cache's calls refuse on the host, without a GPU; and the numpy model's own arithmetic."""
import ctypes as C
import os

import numpy as np
import pytest

from tests import kv_model as M

INVALID, UNSUPPORTED = 1, 2
MEM = 0x10000  # an address that no refused call touches


@pytest.fixture(scope="module")
def jxlib():
    from jxai_amd import _lib
    if not os.path.exists(_lib.LIB_PATH):
        from jxai_amd import build
        build.build(verbose=False)
    return _lib.lib()


def cache(**change):
    from jxai_amd import _lib
    d = _lib.KVCacheDesc(0, 2, 8, 64, 2, 128, 4, 4)
    for name in ("codes", "scales", "table", "len", "ref", "status", "scratch"):
        setattr(d, name, MEM)
    for name, value in change.items():
        setattr(d, name, value)
    return d


def batch(**change):
    from jxai_amd import _lib
    d = _lib.KVBatchDesc(2, 5, 3, 100, MEM, MEM)
    for name, value in change.items():
        setattr(d, name, value)
    return d


def attention(**change):
    from jxai_amd import _lib
    d = _lib.AttentionDesc(8, 0, 0.1, 0.0, 0, 1, 0, 0, None)
    for name, value in change.items():
        setattr(d, name, value)
    return d


SHAPES = [(dict(n_layers=0), INVALID), (dict(n_pages=0), INVALID), (dict(n_kv_heads=0), INVALID), (dict(max_seqs=0), INVALID),
          (dict(max_pages=-1), INVALID), (dict(page_tokens=16), UNSUPPORTED), (dict(page_tokens=96), UNSUPPORTED),
          (dict(page_tokens=512), UNSUPPORTED), (dict(head_dim=16), UNSUPPORTED), (dict(head_dim=80), UNSUPPORTED),
          (dict(head_dim=288), UNSUPPORTED), (dict(n_kv_heads=70000), UNSUPPORTED), (dict(n_pages=2 ** 30), UNSUPPORTED),
          (dict(max_pages=2 ** 25), UNSUPPORTED), (dict(max_seqs=2 ** 20, max_pages=2 ** 12), UNSUPPORTED)]


@pytest.mark.parametrize("change,rc", SHAPES, ids=str)
def test_shapes(jxlib, change, rc):
    c = cache(**change)
    assert jxlib.jx_kv_scratch_words(C.byref(c)) == 0
    assert jxlib.jx_kv_compact(C.byref(c), None) == rc
    assert jxlib.jx_kv_append(C.byref(c), C.byref(batch()), 0, 0, MEM, MEM, 0, None) == rc
    assert jxlib.jx_kv_attention_workspace(C.byref(c), C.byref(batch()), C.byref(attention())) == 0
    assert jxlib.jx_kv_attention(C.byref(c), C.byref(batch()), C.byref(attention()), 0, MEM, MEM, MEM, 1 << 40, None) == rc
    assert jxlib.jx_moe_last_error()


@pytest.mark.parametrize("change", [{n: None} for n in ("codes", "scales", "table", "len", "ref", "status", "scratch")] +
                         [dict(codes=MEM + 8), dict(scales=MEM + 2), dict(table=MEM + 1)], ids=str)
def test_memory(jxlib, change):
    c = cache(**change)
    for call in (lambda: jxlib.jx_kv_reserve(C.byref(c), MEM, None, 1, None), lambda: jxlib.jx_kv_trim(C.byref(c), MEM, None, 1, None),
                 lambda: jxlib.jx_kv_fork(C.byref(c), MEM, MEM, 1, None), lambda: jxlib.jx_kv_compact(C.byref(c), None),
                 lambda: jxlib.jx_kv_append(C.byref(c), C.byref(batch()), 0, 0, MEM, MEM, 0, None),
                 lambda: jxlib.jx_kv_attention(C.byref(c), C.byref(batch()), C.byref(attention()), 0, MEM, MEM, MEM, 1 << 40, None)):
        assert call() == INVALID


def test_lists(jxlib):
    c = cache()
    L = jxlib
    for rc, call in ((INVALID, lambda: L.jx_kv_reserve(None, MEM, None, 1, None)),
                     (INVALID, lambda: L.jx_kv_reserve(C.byref(c), None, None, 1, None)),
                     (INVALID, lambda: L.jx_kv_reserve(C.byref(c), MEM, None, -1, None)),
                     (INVALID, lambda: L.jx_kv_reserve(C.byref(c), MEM, None, 5, None)),
                     (INVALID, lambda: L.jx_kv_reserve(C.byref(c), MEM + 2, None, 1, None)),
                     (INVALID, lambda: L.jx_kv_reserve(C.byref(c), MEM, MEM + 1, 1, None)),
                     (INVALID, lambda: L.jx_kv_trim(C.byref(c), None, None, 2, None)),
                     (INVALID, lambda: L.jx_kv_trim(C.byref(c), MEM, MEM + 3, 2, None)),
                     (INVALID, lambda: L.jx_kv_fork(C.byref(c), MEM, None, 2, None)),
                     (INVALID, lambda: L.jx_kv_fork(C.byref(c), None, MEM, 2, None)),
                     (INVALID, lambda: L.jx_kv_compact(None, None)),
                     (0, lambda: L.jx_kv_reserve(C.byref(c), None, None, 0, None)),
                     (0, lambda: L.jx_kv_fork(C.byref(c), MEM, MEM, 0, None))):
        assert call() == rc


@pytest.mark.parametrize("change", [dict(n_seqs=-1), dict(n_rows=-1), dict(max_rows=-1), dict(max_len=-1), dict(max_rows=6),
                                    dict(row_start=None), dict(row_start=None, n_rows=2, max_rows=0),
                                    dict(seqs=None, n_seqs=5), dict(seqs=MEM + 2), dict(row_start=MEM + 1)], ids=str)
def test_batches(jxlib, change):
    c, b = cache(), batch(**change)
    assert jxlib.jx_kv_append(C.byref(c), C.byref(b), 0, 0, MEM, MEM, 0, None) == INVALID
    assert jxlib.jx_kv_attention(C.byref(c), C.byref(b), C.byref(attention()), 0, MEM, MEM, MEM, 1 << 40, None) == INVALID


def test_append_arguments(jxlib):
    c, b = cache(), batch()
    call = lambda layer=0, t=0, k=MEM, v=MEM, stride=0, bb=b: jxlib.jx_kv_append(C.byref(c), C.byref(bb), layer, t, k, v, stride, None)  # noqa: E731
    assert call(layer=2) == INVALID and call(layer=-1) == INVALID
    assert call(t=8) == UNSUPPORTED
    assert call(k=None) == INVALID and call(v=None) == INVALID
    assert call(k=MEM + 2) == INVALID and call(t=1, v=MEM + 1) == INVALID
    assert call(stride=255) == INVALID and call(stride=-256) == INVALID
    assert call(bb=batch(n_seqs=0)) == 0 and call(bb=batch(max_rows=0)) == 0
    assert jxlib.jx_kv_append(C.byref(c), None, 0, 0, MEM, MEM, 0, None) == INVALID
    assert call(bb=batch(n_seqs=2 ** 30, n_rows=2 ** 20, max_rows=2 ** 20)) == UNSUPPORTED


@pytest.mark.parametrize("change,rc", [(dict(n_heads=0), INVALID), (dict(n_heads=7), INVALID), (dict(type=8), UNSUPPORTED),
                                       (dict(scale=float("nan")), INVALID), (dict(scale=float("inf")), INVALID),
                                       (dict(softcap=-1.0), INVALID), (dict(softcap=float("nan")), INVALID),
                                       (dict(softcap=float("inf")), INVALID), (dict(window=-1), INVALID), (dict(causal=2), INVALID),
                                       (dict(alibi=MEM + 1), INVALID), (dict(q_stride=1023), INVALID), (dict(out_stride=-1024), INVALID)],
                         ids=str)
def test_attention_arguments(jxlib, change, rc):
    c, b, a = cache(), batch(), attention(**change)
    assert jxlib.jx_kv_attention_workspace(C.byref(c), C.byref(b), C.byref(a)) == 0
    assert jxlib.jx_kv_attention(C.byref(c), C.byref(b), C.byref(a), 0, MEM, MEM, MEM, 1 << 40, None) == rc


def test_attention_memory(jxlib):
    from jxai_amd import _lib
    c, a = cache(max_pages=4096), attention()
    b = batch(max_len=0)
    need = jxlib.jx_kv_attention_workspace(C.byref(c), C.byref(b), C.byref(a))
    assert need > 0  # up to 262144 tokens for a few rows: divided
    call = lambda q=MEM, out=MEM, ws=MEM, n=need, layer=0, bb=b: jxlib.jx_kv_attention(C.byref(c), C.byref(bb), C.byref(a), layer, q, out, ws, n, None)  # noqa: E731
    assert call(q=None) == INVALID and call(out=None) == INVALID
    assert call(q=MEM + 2) == INVALID and call(out=MEM + 1) == INVALID
    assert call(ws=None) == INVALID and call(n=need - 1) == INVALID and call(ws=MEM + 4) == INVALID
    assert call(layer=2) == INVALID
    assert call(bb=batch(n_seqs=0)) == 0 and call(bb=batch(max_rows=0)) == 0
    assert jxlib.jx_kv_attention(C.byref(c), C.byref(b), None, 0, MEM, MEM, MEM, need, None) == INVALID
    if not os.path.exists("/dev/kfd"):
        assert call() == 5  # JX_ERR_NODEVICE: everything else was in order
        with pytest.raises(_lib.JxError):
            from jxai_amd import kv
            kv.KVCache(n_layers=1, n_pages=1, page_tokens=32, n_kv_heads=1, head_dim=32, max_seqs=1, max_pages=1)


def test_model_of_append():
    """The plain model against the definition: codes are the nearest integers, scales the largest value's, the layout a bijection."""
    for D in (32, 96, 256):
        for table in (M.k_bytes(D), M.v_bytes(D)):
            assert sorted(table.reshape(-1)) == list(range(32 * D))
    c = M.Cache(1, 4, 32, 1, 32, 1, 3)
    rng = np.random.default_rng(0)
    assert c.reserve([0], [40])
    k, v = rng.standard_normal((2, 40, 1, 32)).astype(np.float32)
    c.append(0, 0, k[:40], v[:40])
    for which, x in ((0, k), (1, v)):
        got = c.tokens(0, 0, which)
        for lo, hi in ((0, 32), (32, 40)):
            step = np.abs(x[lo:hi]).max() / 127
            assert np.abs(got[lo:hi] - x[lo:hi]).max() <= step * (0.5 + 1e-5)
    # a larger value later: earlier codes are at most half an old and half a new step off
    assert c.reserve([0], [1])
    c.append(0, 0, np.full((1, 1, 32), 9, np.float32), np.full((1, 1, 32), 9, np.float32))
    got = c.tokens(0, 0, 0)
    assert np.abs(got[32:40] - k[32:40]).max() <= 0.5 * (9 / 127 + np.abs(k[32:40]).max() / 127) * (1 + 1e-5)
