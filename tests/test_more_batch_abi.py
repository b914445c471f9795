"""The entry points of the cache of 8 bits an element, of the decode with a shared
prefix and of the rules on logits, on the CPU: what they refuse before touching a
device. No kernel is launched."""
import ctypes
import errno

import pytest

import ikv
from test_batch_abi import BAD_BATCHES, P, _batch


def _q8(kc=P, ks=P, vc=P, vs=P, heads=8, dim=128, fmt=0):
    return ctypes.byref(ikv.KvQ8(kc, ks, vc, vs, heads, dim, fmt))


BAD_CACHES = [(None, errno.EINVAL), (dict(heads=0), errno.EINVAL), (dict(dim=0), errno.EINVAL),
              (dict(heads=-1), errno.EINVAL), (dict(fmt=2), errno.EINVAL), (dict(fmt=-1), errno.EINVAL),
              (dict(dim=24), errno.ENOTSUP), (dict(dim=272), errno.ENOTSUP), (dict(dim=100), errno.ENOTSUP),
              (dict(heads=1 << 17), errno.EOVERFLOW)]


def _append(cache="ok", kr=P, vr=P, batch="ok", start=P, first=None, n=10):
    return ikv.load().ikv_append_packed_q8(_q8() if cache == "ok" else cache, kr, vr,
                                           _batch() if batch == "ok" else batch, start, first, n, None)


def _read(cache="ok", kr=P, vr=P, batch="ok", start=P, first=None, n=10):
    return ikv.load().ikv_read_packed_q8(_q8() if cache == "ok" else cache, kr, vr,
                                         _batch() if batch == "ok" else batch, start, first, None, n, None)


def _decode(q=P, cache="ok", batch="ok", n_kv=P, kn=P, vn=P, out=P, n_head=16, ws=P, wsb=1 << 40):
    return ikv.load().ikv_attn_decode_batch_q8(q, _q8() if cache == "ok" else cache,
                                               _batch() if batch == "ok" else batch, n_kv, kn, vn, out, n_head,
                                               0.0, ws, wsb, None)


def _shared(q=P, kp=P, vp=P, batch="ok", start=P, blocks=P, groups=2, n_kv=P, kn=P, vn=P, out=P, n_head=16,
            n_head_kv=8, dim=128, ws=P, wsb=1 << 40):
    return ikv.load().ikv_attn_decode_shared_f32(q, kp, vp, _batch() if batch == "ok" else batch, start, blocks,
                                                 groups, n_kv, kn, vn, out, n_head, n_head_kv, dim, 0.0, ws, wsb,
                                                 None)


@pytest.mark.parametrize("call", [_append, _read, _decode, _shared])
@pytest.mark.parametrize("batch,code", BAD_BATCHES)
def test_a_bad_batch(call, batch, code):
    assert call(batch=None if batch is None else _batch(**batch)) == -code


@pytest.mark.parametrize("call", [_append, _read, _decode])
@pytest.mark.parametrize("cache,code", BAD_CACHES)
def test_a_bad_cache(call, cache, code):
    assert call(cache=None if cache is None else _q8(**cache)) == -code


@pytest.mark.parametrize("call", [_append, _read])
def test_bad_rows(call):
    for name in ("kr", "vr", "start"):
        assert call(**{name: None}) == -errno.EINVAL, name
    for name in ("kr", "vr"):
        assert call(**{name: P + 4}) == -errno.EINVAL, name
    for name in ("kc", "ks", "vc", "vs"):
        assert call(cache=_q8(**{name: None})) == -errno.EINVAL, name
        assert call(cache=_q8(**{name: P + 4})) == -errno.EINVAL, name
    assert call(n=-1) == -errno.EINVAL
    assert call(n=1 << 31) == -errno.EOVERFLOW
    assert call(n=0) == 0 and call(batch=_batch(n_seq=0, tables=None)) == 0  # nothing is launched


def test_bad_decodes():
    for name in ("q", "n_kv", "kn", "vn", "out", "ws"):
        assert _decode(**{name: None}) == -errno.EINVAL, name
    for name in ("q", "kn", "vn", "out", "ws"):
        assert _decode(**{name: P + 4}) == -errno.EINVAL, name
    for name in ("kc", "ks", "vc", "vs"):
        assert _decode(cache=_q8(**{name: None})) == -errno.EINVAL, name
    assert _decode(n_head=12) == -errno.EINVAL and _decode(n_head=0) == -errno.EINVAL
    need = ikv.load().ikv_attn_decode_batch_q8_workspace_bytes(16, 8, 128)
    assert need > 0 and _decode(wsb=need - 1) == -errno.EINVAL
    assert _decode(n_head=1 << 24) == -errno.EOVERFLOW
    assert _decode(batch=_batch(n_seq=0, tables=None, stride=0)) == 0
    size = ikv.load().ikv_attn_decode_batch_q8_workspace_bytes
    for bad in ((12, 8, 128), (0, 8, 128), (16, 8, 0), (16, 8, 264), (16, 8, 20), (16, 0, 128)):
        assert size(*bad) == 0, bad


def test_bad_shared_decodes():
    for name in ("q", "kp", "vp", "n_kv", "kn", "vn", "out", "ws", "start", "blocks"):
        assert _shared(**{name: None}) == -errno.EINVAL, name
    assert _shared(groups=-1) == -errno.EINVAL
    assert _shared(groups=(1 << 20) + 1) == -errno.EOVERFLOW
    assert _shared(n_head=12) == -errno.EINVAL and _shared(n_head=0) == -errno.EINVAL
    assert _shared(dim=0) == -errno.EINVAL and _shared(dim=513) == -errno.ENOTSUP
    assert _shared(ws=P + 4) == -errno.EINVAL
    assert _shared(n_head=1 << 17, n_head_kv=1 << 17) == -errno.EOVERFLOW
    size = ikv.load().ikv_attn_decode_shared_workspace_bytes
    need = size(3, 2, 16, 8, 128)
    assert need > 0 and _shared(wsb=need - 1) == -errno.EINVAL
    assert _shared(batch=_batch(n_seq=0, tables=None)) == 0
    for bad in ((-1, 1, 16, 8, 128), (1, -1, 16, 8, 128), (1, 1, 12, 8, 128), (1, 1, 16, 8, 0), (1, 1, 16, 8, 513),
                ((1 << 20) + 1, 1, 16, 8, 128), (1, (1 << 20) + 1, 16, 8, 128)):
        assert size(*bad) == 0, bad


def test_bad_logit_rules():
    def call(x=P, out=P, n=3, vocab=100, rules=True, **r):
        given = ikv.LogitRules(**{**dict(history=P, history_stride=4, bias_tokens=P, bias_values=P, bias_stride=2,
                                         masks=P, n_masks=1), **r})
        return ikv.load().ikv_adjust_logits_f32(x, out, ctypes.byref(given) if rules else None, n, vocab, None, None)

    assert call(rules=False) == -errno.EINVAL
    assert call(x=None) == -errno.EINVAL and call(out=None) == -errno.EINVAL
    assert call(n=-1) == -errno.EINVAL and call(vocab=0) == -errno.EINVAL and call(vocab=-4) == -errno.EINVAL
    assert call(history_stride=-1) == -errno.EINVAL and call(bias_stride=-1) == -errno.EINVAL
    assert call(bias_values=None) == -errno.EINVAL and call(n_masks=0) == -errno.EINVAL
    big = (1 << 30) + 1
    assert call(vocab=big) == -errno.EOVERFLOW and call(n=(1 << 21) + 1) == -errno.EOVERFLOW
    assert call(n=1 << 21, vocab=1 << 16) == -errno.EOVERFLOW
    assert call(history_stride=big) == -errno.EOVERFLOW and call(bias_stride=big) == -errno.EOVERFLOW
    assert call(n=0) == 0
