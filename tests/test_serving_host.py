"""Refusals of the full-precision scan, the adapters and the sampling that need
no GPU: the C entry points reject bad calls before any launch, the Python
functions reject host tensors."""
import pytest
import torch

from mamba2_recall import _native, adapters, full_state, sampling

FAKE = 1 << 20   # an aligned address that no rejected call reads


def _fails(name, args, text):
    lib = _native.lib()
    assert getattr(lib, name)(*args) != 0
    assert text in lib.m2r_last_error().decode()


def _scan_args(**kw):
    v = dict(x=FAKE, xs_b=8192, xs_l=8192, dt=FAKE, ds_b=128, ds_l=128, A=FAKE, B=FAKE, bs_b=1024, bs_l=1024, C=FAKE,
             cs_b=1024, cs_l=1024, D=FAKE, d32=0, bias=FAKE, b32=0, state=FAKE, pool=4, slots=None, lengths=None, y=FAKE,
             batch=2, L=1, H=128, P=64, G=8, ws=None, ws_bytes=0, stream=None)
    v.update(kw)
    return list(v.values())


@pytest.mark.parametrize("kw,text", [
    (dict(batch=0), "bad geometry"), (dict(L=0), "bad geometry"), (dict(H=-1), "bad geometry"),
    (dict(P=0), "bad geometry"), (dict(G=0), "bad geometry"), (dict(G=7), "bad geometry"), (dict(pool=0), "bad geometry"),
    (dict(batch=(1 << 24) + 1), "size limits"), (dict(L=1 << 25), "size limits"), (dict(P=1 << 25), "size limits"),
    (dict(batch=5), "more batch rows than carries"),
    (dict(x=None), "null pointer"), (dict(dt=None), "null pointer"), (dict(A=None), "null pointer"),
    (dict(B=None), "null pointer"), (dict(C=None), "null pointer"), (dict(D=None), "null pointer"),
    (dict(bias=None), "null pointer"), (dict(state=None), "null pointer"), (dict(y=None), "null pointer"),
    (dict(state=FAKE + 4), "16-byte aligned"),
    (dict(L=512), "workspace too small"), (dict(L=512, ws=FAKE, ws_bytes=64), "workspace too small"),
    (dict(L=512, ws=FAKE + 8, ws_bytes=1 << 40), "not 16-byte aligned")])
def test_scan_rejects(kw, text):
    _fails("m2r_full_scan", _scan_args(**kw), text)


def test_scan_workspace():
    size = _native.lib().m2r_full_scan_workspace
    assert size(1, 1, 128, 64, 8) == 0 and size(64, 2048, 128, 64, 8) == 0   # enough rows without segments
    one = size(1, 2048, 128, 64, 8)
    assert 0 < one <= 256 * 128 * (64 * 128 + 1) * 4
    assert size(1, 8192, 128, 64, 8) == one                                  # segments, not tokens
    assert size(0, 8, 8, 8, 8) == 0 and size(1, 64, 10, 64, 3) == 0


def _adapter_args(**kw):
    v = dict(x=FAKE, xs=64, base=FAKE, bs=32, down=FAKE, up=FAKE, scale=FAKE, ids=FAKE, out=FAKE, os=32, M=4, K=64, N=32,
             n=2, rank=8, ws=FAKE, ws_bytes=1 << 30, stream=None)
    v.update(kw)
    return list(v.values())


@pytest.mark.parametrize("kw,text", [
    (dict(M=0), "non-positive"), (dict(K=0), "non-positive"), (dict(N=-1), "non-positive"), (dict(n=0), "non-positive"),
    (dict(rank=0), "non-positive"), (dict(rank=257), "size limits"), (dict(M=(1 << 24) + 1), "size limits"),
    (dict(x=None), "null pointer"), (dict(base=None), "null pointer"), (dict(down=None), "null pointer"),
    (dict(up=None), "null pointer"), (dict(scale=None), "null pointer"), (dict(ids=None), "null pointer"),
    (dict(out=None), "null pointer"), (dict(ws=None), "null pointer"),
    (dict(down=FAKE + 2), "16-byte aligned"), (dict(up=FAKE + 8), "16-byte aligned"),
    (dict(xs=63), "rows overlap"), (dict(bs=31), "rows overlap"), (dict(os=31), "rows overlap"),
    (dict(ws=FAKE + 4), "workspace"), (dict(ws_bytes=4), "workspace")])
def test_adapters_reject(kw, text):
    _fails("m2r_adapters_add", _adapter_args(**kw), text)


def test_adapters_workspace():
    size = _native.lib().m2r_adapters_workspace
    for rows in (1, 64, 65, 512, 513, 100000):
        n = size(rows, 4096, 4096, 16)
        assert n % (4 * rows * 16) == 0 and 1 <= n // (4 * rows * 16) <= 4
        assert size(rows, 4096, 4096, 9) == n                                # the rank's padding
    assert size(0, 1, 1, 1) == 0


def _sample_args(**kw):
    v = dict(logits=FAKE, dtype=0, stride=1000, u=FAKE, t=None, t_all=1.0, k=None, k_all=0, p=None, p_all=1.0, m=None,
             m_all=0.0, ids=FAKE, lp=FAKE, batch=2, V=1000, ws=FAKE, ws_bytes=1 << 30, stream=None)
    v.update(kw)
    return list(v.values())


@pytest.mark.parametrize("kw,text", [
    (dict(batch=0), "non-positive"), (dict(V=0), "non-positive"), (dict(V=1 << 31), "size limits"),
    (dict(batch=1 << 31), "size limits"), (dict(dtype=3), "binary16"), (dict(dtype=-1), "binary16"),
    (dict(logits=None), "null pointer"), (dict(u=None), "null pointer"), (dict(ids=None), "null pointer"),
    (dict(lp=None), "null pointer"), (dict(stride=999), "rows overlap"), (dict(ws=None), "workspace"),
    (dict(ws=FAKE + 8), "workspace"), (dict(ws_bytes=64), "workspace")])
def test_sample_rejects(kw, text):
    _fails("m2r_sample", _sample_args(**kw), text)


def test_host_tensors_are_refused():
    x = torch.zeros(1, 2, 8, 16, dtype=torch.float16)
    bc, h = torch.zeros(1, 2, 1, 128, dtype=torch.float16), torch.zeros(8)
    state = full_state.allocate_state(1, 8, 16, 128, "cpu")
    with pytest.raises(ValueError, match="x must be CUDA FP16"):
        full_state.scan(x, x[..., 0], h, bc, bc, h, h, state)
    for args in ((1, 8, 16, 64), (0, 8, 16, 128), (1, 0, 16, 128), (1, 8, -1, 128)):
        with pytest.raises(ValueError):
            full_state.allocate_state(*args, "cpu")
    with pytest.raises(ValueError, match="down must be CUDA FP16"):
        adapters.AdapterSet(torch.zeros(1, 8, 16, dtype=torch.float16), torch.zeros(1, 4, 8, dtype=torch.float16))
    with pytest.raises(ValueError, match="AdapterSet"):
        adapters.add(x, x, None, torch.zeros(1, dtype=torch.int32))
    with pytest.raises(ValueError, match="logits must be CUDA"):
        sampling.sample(torch.zeros(1, 10), torch.zeros(1))
    with pytest.raises(ValueError, match="logits must be CUDA"):
        sampling.sample([1.0], torch.zeros(1))
