"""Sizes of the sampling's workspace, on the host."""
import pytest

from mamba2_recall import _native


def test_no_larger_than_the_call_needs():
    lib = _native.lib()
    whole, call = lib.m2r_sample_workspace, lib.m2r_sample_call_workspace
    assert whole(0, 1000) == 0 and call(0, 1000, 0, 1.0, 0, 1.0) == 0
    # the cut's list holds no more than a row's tokens, and 4,096 of them
    assert whole(7, 500) - whole(7, 100) == 7 * 8 * 400
    assert whole(1, 4096) == whole(1, 256000)
    for vocab in (1, 500, 256000):
        plain = call(64, vocab, 0, 1.0, 0, 1.0)
        assert plain <= 64 * 4352 and plain % 128 == 0                # units, ranges and counters
        assert whole(64, vocab) - plain >= 64 * 6144                  # the bins
        assert call(64, vocab, 0, 0.7, vocab, 1.0) == plain           # a top-k of the whole row
        for kw in ((1, 1.0, 0, 1.0), (0, 0.0, 0, 1.0), (0, 1.0, 0, 0.9)) + (((0, 1.0, 1, 1.0),) if vocab > 1 else ()):
            assert call(64, vocab, *kw) == whole(64, vocab), kw
    assert whole(4096, 500) <= 65 << 20


@pytest.mark.parametrize("filters,size", [(dict(), 0), (dict(k_all=50), 1), (dict(p_all=0.5), 1), (dict(t_all=0.0), 1)])
def test_call_checks_what_it_needs(filters, size):
    """One byte less than the call's own size is refused before any launch."""
    v = dict(logits=1 << 20, dtype=0, stride=1000, u=1 << 20, t=None, t_all=1.0, k=None, k_all=0, p=None, p_all=1.0, m=None,
             m_all=0.0, ids=1 << 20, lp=1 << 20, batch=2, V=1000, ws=1 << 20, ws_bytes=0, stream=None)
    v.update(filters)
    lib = _native.lib()
    need = lib.m2r_sample_call_workspace(2, 1000, 0, v["t_all"], v["k_all"], v["p_all"])
    assert (need == lib.m2r_sample_workspace(2, 1000)) == bool(size)
    v["ws_bytes"] = need - 1
    assert lib.m2r_sample(*v.values()) != 0 and "workspace" in lib.m2r_last_error().decode()
