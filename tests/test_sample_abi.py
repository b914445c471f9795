"""ikv_sample_f32 on the CPU: what it refuses before touching a device."""
import errno

import ikv

P = 4096  # a non-null, aligned "device" address; never dereferenced


def _sample(logits=P, u=P, t=None, k=None, p=None, m=None, rows=3, vocab=1000, token=P, logprob=None,
            ws=P, wsb=1 << 50):
    return ikv.load().ikv_sample_f32(logits, u, t, k, p, m, rows, vocab, token, logprob, ws, wsb, None)


def test_sample_refuses_bad_arguments():
    for name in ("logits", "u", "token", "ws"):
        assert _sample(**{name: None}) == -errno.EINVAL, name
    assert _sample(rows=-1) == -errno.EINVAL
    assert _sample(vocab=0) == -errno.EINVAL
    assert _sample(vocab=-5) == -errno.EINVAL
    assert _sample(vocab=(1 << 30) + 1) == -errno.EOVERFLOW
    assert _sample(rows=(1 << 21) + 1) == -errno.EOVERFLOW
    assert _sample(ws=P + 4) == -errno.EINVAL
    need = ikv.load().ikv_sample_workspace_bytes(3, 1000)
    assert need > 0 and _sample(wsb=need - 1) == -errno.EINVAL
    assert _sample(rows=0) == 0  # nothing is launched


def test_sample_workspace_of_no_rows():
    size = ikv.load().ikv_sample_workspace_bytes
    assert size(0, 10) == 0 and size(10, 0) == 0 and size(-1, 10) == 0


def test_sample_workspace_is_enough_for_fewer_rows():
    size = ikv.load().ikv_sample_workspace_bytes
    for vocab in (10, 16384, 16385, 151936):
        sizes = [size(rows, vocab) for rows in range(1, 1200)]
        assert sizes == sorted(sizes)
