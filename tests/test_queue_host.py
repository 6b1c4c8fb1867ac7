"""Refusals of the 8-bit projections, the adjusted logits and the ragged
convolution that need no GPU: the C entry points reject bad calls before any
launch, the Python functions reject host tensors, generate() bad settings
before it touches the request."""
import pytest
import torch

from mamba2_recall import _native, full_state, int8, sampling
from mamba2_recall.generate import generate

FAKE = 1 << 20   # an aligned address that no rejected call reads


def _fails(name, args, text):
    lib = _native.lib()
    assert getattr(lib, name)(*args) != 0
    assert text in lib.m2r_last_error().decode()


def _linear_args(**kw):
    v = dict(x=FAKE, x_dtype=0, xs=256, w=FAKE, ws=FAKE, y=FAKE, y_dtype=0, ys=512, M=3, N=512, K=256, work=FAKE,
             work_bytes=1 << 40, stream=None)
    v.update(kw)
    return list(v.values())


@pytest.mark.parametrize("kw,text", [
    (dict(M=0), "non-positive"), (dict(N=0), "non-positive"), (dict(K=-1), "non-positive"),
    (dict(M=(1 << 24) + 1), "size limits"), (dict(N=(1 << 24) + 1), "size limits"), (dict(K=131073), "size limits"),
    (dict(ys=(1 << 25) + 1), "size limits"), (dict(x_dtype=2), "x must be"), (dict(x_dtype=-1), "x must be"),
    (dict(y_dtype=3), "y must be"), (dict(x=None), "null pointer"), (dict(w=None), "null pointer"),
    (dict(ws=None), "null pointer"), (dict(y=None), "null pointer"), (dict(xs=-1), "negative stride"),
    (dict(ys=511), "rows overlap"), (dict(w=FAKE + 8), "16-byte aligned"),
    (dict(M=64, work=None), "workspace"), (dict(M=64, work=FAKE + 4), "workspace"), (dict(M=64, work_bytes=64), "workspace"),
    (dict(x=FAKE + 2, work=None), "workspace")])
def test_int8_linear_rejects(kw, text):
    _fails("m2r_int8_linear", _linear_args(**kw), text)


@pytest.mark.parametrize("kw,text", [
    (dict(N=0), "non-positive"), (dict(K=0), "non-positive"), (dict(K=1 << 18), "size limits"), (dict(dtype=2), "weights must be"),
    (dict(w=None), "null pointer"), (dict(tiles=None), "null pointer"), (dict(scale=None), "null pointer"),
    (dict(ws=-4), "negative stride"), (dict(tiles=FAKE + 4), "16-byte aligned")])
def test_int8_quantize_rejects(kw, text):
    v = dict(w=FAKE, dtype=0, ws=256, tiles=FAKE, scale=FAKE, N=8, K=256, stream=None)
    v.update(kw)
    _fails("m2r_int8_quantize", list(v.values()), text)


def test_int8_sizes():
    lib = _native.lib()
    assert lib.m2r_int8_weight_bytes(1, 1) == 32 * 128 and lib.m2r_int8_weight_bytes(33, 129) == 64 * 256
    assert lib.m2r_int8_weight_bytes(18560, 4096) == 18560 * 4096 and lib.m2r_int8_weight_bytes(0, 5) == 0
    need = lib.m2r_int8_linear_workspace
    assert need(FAKE, 4096, 4, 18560, 4096) == 0                 # codes formed in the product's launch
    assert need(FAKE + 2, 4096, 4, 18560, 4096) > 0 and need(FAKE, 4095, 4, 18560, 4096) > 0
    assert need(FAKE, 8208, 1, 64, 8208) > 0
    assert need(FAKE, 4096, 2048, 18560, 4096) == 2048 * 4096 + 4 * 2048
    assert need(FAKE, 8192, 192, 4096, 8192) > 192 * 8192        # and the sums of split inputs
    assert need(FAKE, 8, 0, 8, 8) == 0


def _adjust_args(**kw):
    v = dict(logits=FAKE, dtype=2, ls=1000, out=FAKE, os=1000, prompt=None, p64=1, ps=0, pn=0, pl=None, tokens=None, t64=1,
             ts=0, tn=0, tl=None, r=None, r_all=1.0, p=None, p_all=0.0, f=None, f_all=0.0, bi=None, bis=0, bv=None, bvs=0,
             n=0, allowed=None, as_=0, masks=0, rows=None, batch=2, V=1000, stream=None)
    v.update(kw)
    return list(v.values())


@pytest.mark.parametrize("kw,text", [
    (dict(batch=0), "non-positive"), (dict(V=0), "non-positive"), (dict(V=1 << 31), "size limits"),
    (dict(batch=1 << 31), "size limits"), (dict(dtype=3), "binary16"), (dict(dtype=-1), "binary16"),
    (dict(logits=None), "null pointer"), (dict(out=None), "null pointer"), (dict(ls=999), "rows overlap"),
    (dict(os=999), "rows overlap"), (dict(pn=-1), "list limits"), (dict(tn=(1 << 30) + 1), "list limits"),
    (dict(n=-1), "list limits"), (dict(pn=4), "null pointer"), (dict(tn=4), "null pointer"), (dict(n=4, bi=FAKE), "null pointer"),
    (dict(ps=-1), "negative strides"), (dict(bvs=-1), "negative strides"), (dict(as_=-1), "negative strides"),
    (dict(allowed=FAKE), "no masks"), (dict(allowed=FAKE, masks=1), "more batch rows than masks")])
def test_adjust_rejects(kw, text):
    _fails("m2r_adjust_logits", _adjust_args(**kw), text)


def _conv_args(**kw):
    v = dict(window=FAKE, pool=4, ws_s=400, ws_t=100, value=FAKE, vs_b=700, vs_l=100, weight=FAKE, bias=None, slots=None,
             lengths=None, x=FAKE, bm=FAKE, cm=FAKE, n_x=80, n_b=10, n_c=10, batch=2, tokens=7, width=4, silu=1, stream=None)
    v.update(kw)
    return list(v.values())


@pytest.mark.parametrize("kw,text", [
    (dict(pool=0), "non-positive"), (dict(n_x=0), "non-positive"), (dict(n_b=-1), "non-positive"), (dict(n_c=0), "non-positive"),
    (dict(batch=0), "non-positive"), (dict(tokens=0), "non-positive"), (dict(width=3), "width must be 4"),
    (dict(tokens=(1 << 24) + 1), "size limits"), (dict(pool=(1 << 24) + 1), "size limits"),
    (dict(window=None), "null pointer"), (dict(value=None), "null pointer"), (dict(weight=None), "null pointer"),
    (dict(x=None), "null pointer"), (dict(bm=None), "null pointer"), (dict(cm=None), "null pointer"),
    (dict(batch=5), "more batch rows than windows"), (dict(ws_t=99), "windows overlap"), (dict(ws_s=399), "windows overlap"),
    (dict(vs_b=-1), "negative strides"), (dict(vs_l=-1), "negative strides"), (dict(weight=FAKE + 4), "8-byte aligned")])
def test_conv_rejects(kw, text):
    _fails("m2r_conv_pool", _conv_args(**kw), text)


def test_host_tensors_are_refused():
    half = torch.zeros(2, 3, 32, dtype=torch.float16)
    with pytest.raises(ValueError, match="value must be CUDA"):
        full_state.convolve(half, torch.zeros(32, 4).half(), None, full_state.allocate_windows(2, 32, "cpu"), (16, 8, 8))
    window = full_state.allocate_windows(3, 32, "cpu")
    assert window.shape == (3, 32, 4) and window.stride() == (128, 1, 32) and window.dtype == torch.float16
    for args in ((0, 8), (4, 0), (-1, 8)):
        with pytest.raises(ValueError):
            full_state.allocate_windows(*args, "cpu")
    with pytest.raises(ValueError, match="codes must be CUDA"):
        int8.Int8Weight(torch.zeros(4, 8, dtype=torch.int8), torch.ones(4))
    with pytest.raises(ValueError, match="weight must be CUDA"):
        int8.Int8Weight.quantize(torch.zeros(4, 8).half())
    with pytest.raises(ValueError, match="Int8Weight"):
        int8.linear(half, None)
    for logits in (torch.zeros(1, 10), [1.0], None):
        with pytest.raises(ValueError, match="logits must be CUDA"):
            sampling.adjust(logits)


class _Controller:
    """A controller that must not be reached."""
    def backbone(self, *args, **kw):
        raise AssertionError("the request was reset")


@pytest.mark.parametrize("kw", [
    dict(repetition=0.0), dict(repetition=-1.0), dict(repetition=True), dict(repetition=torch.ones(2)),
    dict(repetition=torch.ones(3, dtype=torch.float64)), dict(presence="x"), dict(frequency=torch.ones(3, dtype=torch.int32)),
    dict(bias=torch.ones(3)), dict(bias=(torch.ones(3), torch.ones(3))), dict(bias=(torch.ones(2, dtype=torch.int32), torch.ones(3))),
    dict(bias=(torch.ones(2, 4, dtype=torch.int32), torch.ones(2, 4))), dict(bias=(torch.ones((), dtype=torch.int32), torch.ones(()))),
    dict(allowed=[1, 2]), dict(allowed=7), dict(lengths=[1, 2, 3]), dict(lengths=torch.ones(3)),
    dict(lengths=torch.ones(2, dtype=torch.int32)), dict(lengths=torch.ones(3, dtype=torch.int64)),
    dict(lengths=torch.ones(3, dtype=torch.int32, device="meta"))])
def test_generate_settings(kw):
    with pytest.raises(ValueError):
        generate(_Controller(), None, torch.zeros(3, 4, dtype=torch.long), torch.zeros(3, 2), **kw)


def test_masks_and_lists_of_the_wrong_shape():
    """The checks behind adjust, on any device."""
    like = torch.zeros(3, 40)
    for allowed, rows in ((torch.zeros(3, dtype=torch.int32), None), (torch.zeros(2, 2, dtype=torch.int32), None),
                          (torch.zeros(3, 2), None), (torch.zeros(0, 2, dtype=torch.int32), None),
                          (torch.zeros(2, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)),
                          (torch.zeros(2, 2, dtype=torch.int32), torch.zeros(3)),
                          (torch.zeros(2, 2, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)),
                          (None, torch.zeros(3, dtype=torch.int32))):
        with pytest.raises(ValueError):
            sampling.masks(like, 40, allowed, rows)
    one, rows = sampling.masks(like, 40, torch.zeros(2, dtype=torch.int32), None)
    assert one.shape == (3, 2) and rows is None
    for ids, lengths in ((torch.zeros(2, 4, dtype=torch.int64), None), (torch.zeros(3, 4), None), (torch.zeros(3, dtype=torch.int32), None),
                         (torch.zeros(3, 4, dtype=torch.int32), torch.zeros(3)), (None, torch.zeros(3, dtype=torch.int32)),
                         (torch.zeros(3, 4, dtype=torch.int32), torch.zeros(4, dtype=torch.int32))):
        with pytest.raises(ValueError):
            sampling._list(ids, lengths, "prompt", 3, -1)


@pytest.mark.parametrize("name,args,text", [
    ("m2r_int8_linear", _linear_args(M=1 << 24, K=16, xs=16, N=1, ys=1), "size limits"),
    ("m2r_int8_linear", _linear_args(M=1 << 22, K=16, xs=16, N=1 << 18, ys=1 << 18, work_bytes=1 << 50), "grid limits"),
    ("m2r_int8_quantize", [FAKE, 0, 16, FAKE, FAKE, (1 << 24) - 127, 16, None], "size limits"),
    ("m2r_adjust_logits", _adjust_args(V=1, ls=1, os=1, batch=1 << 24), "grid limits"),
    ("m2r_adjust_logits", _adjust_args(batch=1 << 23, tokens=FAKE, tn=8192), "grid limits"),
    ("m2r_conv_pool", _conv_args(batch=8, pool=8, n_x=1, n_b=1, n_c=1, tokens=1 << 24), "grid limits"),
    ("m2r_conv_pool", _conv_args(batch=1 << 24, pool=1 << 24, tokens=1), "grid limits")])
def test_launches_of_2_to_the_32_threads_are_refused(name, args, text):
    """A launch has fewer than 2^32 threads: calls that would need more are refused before it."""
    _fails(name, args, text)


def test_padding_is_never_looked_up():
    """Ids behind a row's length, of any value, do not reach the embedding: one
    outside the vocabulary would end a process there."""
    from types import SimpleNamespace
    class OnHost(full_state.FullState):
        device, _installed = torch.device("cpu"), True
    c = OnHost.__new__(OnHost)
    seen = []
    c._running, c._adapters = False, None
    c._request = SimpleNamespace(next_layer=0, failed=False)
    c.model = SimpleNamespace(backbone=lambda ids: seen.append(ids) or torch.nn.functional.embedding(ids, torch.zeros(50, 8)))
    ids = torch.tensor([[7, 8, 9, -1], [3, -1, -1, -1], [4, 5, 6, 7], [1 << 40, -100, 50, 99]])
    given = ids.clone()
    c.backbone(ids, lengths=torch.tensor([3, 1, 9, -2], dtype=torch.int32))
    assert seen[0].tolist() == [[7, 8, 9, 0], [3, 0, 0, 0], [4, 5, 6, 7], [0, 0, 0, 0]] and torch.equal(ids, given)
    c.backbone(ids[2:3])
    assert seen[1].tolist() == [[4, 5, 6, 7]]
