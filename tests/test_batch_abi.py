"""The entry points of a step over several sequences (include/ikv_batch.h) on
the CPU: what they refuse before touching a device. No kernel is launched."""
import ctypes
import errno

import pytest

import ikv

P = 4096  # a non-null, 16-byte aligned "device" address; never dereferenced


def _batch(tables=P, stride=4, bt=64, pool=8, n_seq=3, status=None):
    return ctypes.byref(ikv.KvBatch(tables, stride, bt, pool, n_seq, status))


BAD_BATCHES = [
    (None, errno.EINVAL),
    (dict(tables=None), errno.EINVAL),
    (dict(stride=0), errno.EINVAL), (dict(stride=-1), errno.EINVAL),
    (dict(bt=0), errno.EINVAL), (dict(bt=32), errno.EINVAL), (dict(bt=-64), errno.EINVAL),
    (dict(bt=100), errno.EINVAL),
    (dict(pool=0), errno.EINVAL), (dict(n_seq=-1), errno.EINVAL),
    (dict(pool=1 << 26), errno.EOVERFLOW),            # 2^32 pool rows
    (dict(n_seq=(1 << 20) + 1), errno.EOVERFLOW),
    (dict(stride=(1 << 22) + 1), errno.EOVERFLOW),    # past 2^28 tokens of a sequence
]


def _append(kp=P, vp=P, kr=P, vr=P, batch="ok", start=P, first=None, n=10, row_bytes=4096):
    b = _batch() if batch == "ok" else batch
    return ikv.load().ikv_append_packed_f32(kp, vp, kr, vr, b, start, first, n, row_bytes, None)


@pytest.mark.parametrize("batch,code", BAD_BATCHES)
def test_append_packed_refuses_a_bad_batch(batch, code):
    assert _append(batch=None if batch is None else _batch(**batch)) == -code


def test_append_packed_refuses_bad_arguments():
    for name in ("kp", "vp", "kr", "vr", "start"):
        assert _append(**{name: None}) == -errno.EINVAL, name
    for name in ("kp", "vp", "kr", "vr"):
        assert _append(**{name: P + 2}) == -errno.EINVAL, name
    assert _append(row_bytes=6) == -errno.EINVAL
    assert _append(n=-1) == -errno.EINVAL
    assert _append(n=1 << 31) == -errno.EOVERFLOW
    # nothing to do: nothing is launched
    assert _append(n=0) == 0
    assert _append(row_bytes=0) == 0
    assert _append(batch=_batch(n_seq=0)) == 0


def _packed(q=P, k=P, v=P, start=P, n_seq=3, n=10, out=P, n_head=16, n_head_kv=8, dim=128):
    return ikv.load().ikv_attn_prefill_packed_f32(q, k, v, start, n_seq, n, out, n_head, n_head_kv, dim,
                                                  0.0, None, None)


def _packed_paged(q=P, k=P, v=P, batch="ok", start=P, past=None, n=10, out=P, n_head=16, n_head_kv=8,
                  dim=128, ws=None, wsb=0):
    b = _batch() if batch == "ok" else batch
    return ikv.load().ikv_attn_prefill_packed_paged_f32(q, k, v, b, start, past, n, out, n_head,
                                                        n_head_kv, dim, 0.0, ws, wsb, None)


@pytest.mark.parametrize("batch,code", BAD_BATCHES)
def test_packed_prefill_refuses_a_bad_batch(batch, code):
    assert _packed_paged(batch=None if batch is None else _batch(**batch)) == -code


@pytest.mark.parametrize("call", [_packed, _packed_paged])
def test_packed_prefill_refuses_bad_arguments(call):
    for name in ("q", "k", "v", "start", "out"):
        assert call(**{name: None}) == -errno.EINVAL, name
    assert call(n_head=12) == -errno.EINVAL  # not a multiple of n_head_kv
    assert call(n_head=0) == -errno.EINVAL
    assert call(n_head_kv=0) == -errno.EINVAL
    assert call(dim=0) == -errno.EINVAL
    assert call(dim=513) == -errno.ENOTSUP
    assert call(n=-1) == -errno.EINVAL
    assert call(n=1 << 24) == -errno.EOVERFLOW
    assert call(n=0) == 0  # nothing is launched
    if call is _packed:
        assert call(n_seq=-1) == -errno.EINVAL
        assert call(n_seq=(1 << 20) + 1) == -errno.EOVERFLOW
        assert call(n_seq=1 << 20, n=1, n_head=4096, n_head_kv=4096) == -errno.EOVERFLOW  # 2^32 blocks
        assert call(n_seq=0) == 0
    else:
        assert call(ws=P + 4, wsb=1 << 30) == -errno.EINVAL
        assert call(n=1, batch=_batch(n_seq=1 << 20, stride=1), n_head=4096, n_head_kv=4096) == -errno.EOVERFLOW


def test_packed_prefill_workspace():
    size = ikv.load().ikv_attn_prefill_packed_paged_workspace_bytes
    assert size(1, 16, 4096, 16, 8, 128) > 0            # few rows, perhaps behind many keys
    assert size(1, 16, 512, 16, 8, 128) == 0            # a table of two parts' keys
    assert size(8, 1 << 16, 1 << 16, 32, 8, 128) == 0   # blocks enough for the card
    assert size(1, 16, 4096, 16, 8, 200) == 0           # the generic kernel's
    assert size(0, 16, 4096, 16, 8, 128) == 0 and size(1, 0, 4096, 16, 8, 128) == 0
    assert size(1, 16, 4096, 12, 8, 128) == 0 and size(1, 16, 1 << 29, 16, 8, 128) == 0


def _decode(q=P, kp=P, vp=P, batch="ok", n_kv=P, kn=P, vn=P, out=P, n_head=16, n_head_kv=8, dim=128,
            ws=P, wsb=1 << 40):
    b = _batch() if batch == "ok" else batch
    return ikv.load().ikv_attn_decode_batch_f32(q, kp, vp, b, n_kv, kn, vn, out, n_head, n_head_kv, dim,
                                                0.0, ws, wsb, None)


@pytest.mark.parametrize("batch,code", BAD_BATCHES)
def test_decode_batch_refuses_a_bad_batch(batch, code):
    assert _decode(batch=None if batch is None else _batch(**batch)) == -code


def test_decode_batch_refuses_bad_arguments():
    for name in ("q", "kp", "vp", "n_kv", "kn", "vn", "out", "ws"):
        assert _decode(**{name: None}) == -errno.EINVAL, name
    assert _decode(n_head=12) == -errno.EINVAL  # not a multiple of n_head_kv
    assert _decode(n_head=0) == -errno.EINVAL
    assert _decode(dim=0) == -errno.EINVAL
    assert _decode(dim=513) == -errno.ENOTSUP
    assert _decode(ws=P + 4) == -errno.EINVAL
    need = ikv.load().ikv_attn_decode_batch_workspace_bytes(16, 8, 128)
    assert need > 0 and _decode(wsb=need - 1) == -errno.EINVAL
    assert _decode(n_head=1 << 17, n_head_kv=1 << 17) == -errno.EOVERFLOW
    assert _decode(batch=_batch(n_seq=0)) == 0  # nothing is launched


def test_decode_batch_workspace_of_refused_shapes():
    size = ikv.load().ikv_attn_decode_batch_workspace_bytes
    assert size(12, 8, 128) == 0 and size(0, 8, 128) == 0 and size(16, 8, 0) == 0 and size(16, 8, 513) == 0


@pytest.mark.parametrize("empty", [dict(tables=None), dict(tables=None, stride=0), dict(stride=0)],
                         ids=lambda e: "+".join(e))
def test_no_sequences_need_no_tables(empty):
    """A step in which nobody is active: an empty table has no address and may have
    no columns."""
    b = _batch(n_seq=0, **empty)
    assert _append(batch=b) == 0
    assert _packed_paged(batch=b) == 0 and _packed_paged(batch=b, past=P) == 0
    assert _decode(batch=b) == 0


def test_no_sequences_are_no_excuse():
    """What else is wrong with a call is refused all the same."""
    for bad in (dict(stride=-1), dict(bt=32), dict(bt=0), dict(pool=0)):
        b = _batch(n_seq=0, **bad)
        assert _append(batch=b) == _packed_paged(batch=b) == _decode(batch=b) == -errno.EINVAL, bad
