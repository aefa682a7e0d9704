"""What the streaming operators refuse, on the CPU: host tensors, and bad arguments at the C boundary (which returns
before it touches a pointer)."""
import copy
import ctypes
import pickle
import types

import pytest
import torch
import torch.autograd.forward_ad as fwd

from oracle import streaming as O
from vasc_amd import _lib, ops
from vasc_amd.streaming import AggregatorStream, BlockCache, stream_attention

FAKE = 1 << 20  # an aligned address that nothing reads


def _rotary(**kw):
    a = dict(q=FAKE, Hq=2, k=None, ko=None, Hk=0, B=1, T=4, D=64, pos=FAKE, axes=3, sections=(16, 24, 24), freq=FAKE,
             dtype=0, qst=64)
    a.update(kw)
    sec = (ctypes.c_int64 * max(1, len(a["sections"])))(*a["sections"])
    _lib.call("vasc_rotary_axes", a["q"], 512, 256, a["qst"], FAKE, 512, 256, 64, a["Hq"], a["k"], 0, 0, 0, a["ko"], 0, 0, 0,
              a["Hk"], a["B"], a["T"], a["D"], a["pos"], 12, 3, a["axes"], ctypes.cast(sec, ctypes.c_void_p), a["freq"],
              a["dtype"], 0, None)


@pytest.mark.parametrize("kw,match", [
    (dict(q=None), "required"), (dict(pos=None), "required"), (dict(freq=None), "required"), (dict(k=FAKE), "together"),
    (dict(B=0), "empty"), (dict(T=0), "empty"), (dict(Hq=0), "empty"), (dict(D=0), "outside"), (dict(D=257), "outside"),
    (dict(axes=0), "axes"), (dict(axes=5), "axes"), (dict(sections=(15, 24, 24)), "even"),
    (dict(sections=(0, 24, 24)), "even"), (dict(sections=(32, 24, 24)), "hold"), (dict(dtype=3), "dtype"),
])
def test_rotary_refuses(kw, match):
    with pytest.raises(_lib.VascError, match=match):
        _rotary(**kw)


def _write(name="vasc_cache_write", **kw):
    a = dict(k=FAKE, st=64, B=1, H=2, T=4, D=64, dtype=0, table=FAKE, ts=8, mp=8, start=FAKE, kc=FAKE, pages=9)
    a.update(kw)
    if name == "vasc_cache_write":
        _lib.call(name, a["k"], 512, 256, a["st"], FAKE, 512, 256, 64, a["B"], a["H"], a["T"], a["D"], a["dtype"],
                  a["table"], a["ts"], a["mp"], a["start"], None, a["kc"], FAKE, FAKE, FAKE, FAKE, a["pages"], None)
    else:
        _lib.call(name, a["kc"], FAKE, FAKE, FAKE, a["pages"], a["table"], a["ts"], a["mp"], a["start"], None, a["B"],
                  a["H"], a["T"], a["D"], a["dtype"], a["k"], FAKE, None)


@pytest.mark.parametrize("name", ["vasc_cache_write", "vasc_cache_read"])
@pytest.mark.parametrize("kw,match", [
    (dict(k=None), "NULL"), (dict(table=None), "required"), (dict(start=None), "required"), (dict(kc=None), "required"),
    (dict(B=0), "empty"), (dict(T=0), "empty"), (dict(D=80), "not built"), (dict(dtype=7), "dtype"),
    (dict(pages=0), "positive"), (dict(mp=0), "positive"), (dict(mp=1 << 24, ts=1 << 24), "too large"),
    (dict(ts=4), "table_stride"), (dict(k=FAKE + 8), "aligned"), (dict(kc=FAKE + 4), "aligned"),
    (dict(T=1 << 30), "too many"), (dict(B=1 << 24), "too many"), (dict(B=1 << 20, T=1 << 20), "too many"),
])
def test_write_and_read_refuse(name, kw, match):
    with pytest.raises(_lib.VascError, match=match):
        _write(name, **kw)


def test_write_refuses_odd_strides():
    with pytest.raises(_lib.VascArgumentError, match="multiples of 8"):
        _write(st=65)


def _select(**kw):
    a = dict(q=FAKE, B=1, Hq=4, H=2, T=8, D=64, dtype=0, mean=FAKE, mp=8, lengths=FAKE, block_q=4, sink=1, recent=1,
             keep=2, causal=0, width=4)
    a.update(kw)
    _lib.call("vasc_cache_select", a["q"], 512, 64, 256, a["B"], a["Hq"], a["H"], a["T"], a["D"], a["dtype"], a["mean"], 9,
              FAKE, a["mp"], a["mp"], a["lengths"], None, a["block_q"], a["sink"], a["recent"], a["keep"], a["causal"],
              FAKE, FAKE, a["width"], FAKE, None)


@pytest.mark.parametrize("kw,match", [
    (dict(q=None), "NULL"), (dict(mean=None), "required"), (dict(lengths=None), "required"), (dict(Hq=5), "multiple"),
    (dict(Hq=0), "multiple"), (dict(dtype=2), "dtype"), (dict(block_q=0), "rows"), (dict(block_q=65), "rows"),
    (dict(Hq=512), "rows"), (dict(recent=0), "recent"), (dict(keep=-1), "negative"), (dict(sink=-1), "negative"),
    (dict(width=5), "width"), (dict(causal=1), "width"), (dict(mp=40000), "not built"), (dict(D=32), "not built"),
    (dict(B=1 << 23, H=2, T=1 << 20), "too many"),
])
def test_select_refuses(kw, match):
    with pytest.raises(_lib.VascError, match=match):
        _select(**kw)


def _attn(**kw):
    a = dict(q=FAKE, o=FAKE, B=1, Hq=4, H=2, T=1, D=64, dtype=0, kc=FAKE, mp=5000, ts=5000, lengths=FAKE, block_q=1,
             index=None, width=0, count=None, ws=None, bytes=0, qst=256, ost=256)
    a.update(kw)
    _lib.call("vasc_cache_attn", a["q"], 512, 64, a["qst"], a["o"], 512, 64, a["ost"], a["B"], a["Hq"], a["H"], a["T"],
              a["D"], a["dtype"], a["kc"], FAKE, FAKE, FAKE, 9, FAKE, a["ts"], a["mp"], a["lengths"], None, a["block_q"],
              a["index"], a["width"], a["count"], 0, 0.125, a["ws"], a["bytes"], None)


@pytest.mark.parametrize("kw,match", [
    (dict(q=None), "NULL"), (dict(kc=None), "NULL"), (dict(lengths=None), "NULL"), (dict(D=96), "not built"),
    (dict(dtype=2), "dtype"), (dict(index=FAKE), "together"), (dict(index=FAKE, count=FAKE), "together"),
    (dict(width=3), "together"), (dict(Hq=3), "sizes"), (dict(block_q=65), "sizes"), (dict(T=0), "sizes"),
    (dict(B=1 << 24), "sizes"), (dict(q=FAKE + 2), "aligned"), (dict(o=FAKE + 4), "aligned"), (dict(qst=260), "multiples"),
    (dict(ost=258), "multiples"), (dict(ts=7), "table_stride"), (dict(), "workspace"), (dict(ws=FAKE, bytes=64), "workspace"),
])
def test_attn_refuses(kw, match):
    with pytest.raises(_lib.VascError, match=match):
        _attn(**kw)


def test_workspace_query():
    size = _lib.fn("vasc_cache_attn_workspace_size")
    assert size(1, 4, 2, 1, 64, 1, 5000, 0) > 0
    assert size(1, 4, 2, 1, 64, 1, 5000, 4) == 0  # a short list is not split
    for bad in ((0, 4, 2, 1, 64, 1, 10, 0), (1, 5, 2, 1, 64, 1, 10, 0), (1, 4, 2, 1, 60, 1, 10, 0), (1, 4, 2, 1, 64, 0, 10, 0),
                (1, 4, 2, 1, 64, 65, 10, 0), (1, 4, 2, 1, 64, 1, 0, 0), (1, 4, 2, 1, 64, 1, 10, -1)):
        assert size(*bad) == -1


def test_host_tensors_are_refused():
    x, i = torch.zeros(1, 2, 4, 64), torch.zeros(1, dtype=torch.int32)
    table = torch.zeros(1, 4, dtype=torch.int32)
    with pytest.raises(ValueError, match="GPU"):
        ops.rotary_axes(x, None, torch.zeros(1, 4, 1, dtype=torch.int32), (16,), torch.zeros(8, dtype=torch.float64))
    for call in (lambda: ops.cache_write(None, x, x, table, i), lambda: ops.cache_read(None, table, i, 4),
                 lambda: ops.cache_select(x, None, table, i, 4), lambda: ops.cache_attn(x, None, table, i)):
        with pytest.raises(ValueError, match="GPU"):
            call()
    with pytest.raises(ValueError, match="GPU"):
        BlockCache(4, 2, 64, device="cpu")
    with pytest.raises(ValueError, match="not built"):
        BlockCache(4, 2, 96)
    with pytest.raises(ValueError, match="pages"):
        BlockCache(0, 2, 64)


def test_captured_call_on_leaves_of_an_eager_graph(monkeypatch):
    """The mark lives as long as the eager graph does, whichever of its tensors is let go first."""
    capturing = [False]
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing[0])
    a, b = torch.ones(2, requires_grad=True), torch.ones(2, requires_grad=True)

    def call(*leaves):
        out = sum(leaves[1:], leaves[0] * 1)  # a graph over all of them
        node = torch.cat(leaves).grad_fn
        ops._one_graph(node)
        return out, node

    eager = call(a)
    capturing[0] = True
    call(b)
    with pytest.raises(ValueError, match="eager graph"):
        call(a, b)
    eager = eager[0]  # the other node goes, the leaf's stays
    with pytest.raises(ValueError, match="eager graph"):
        call(a)
    del eager
    call(a, b)


def test_copied_cache_has_addresses_of_its_own(tmp_path):
    """A copy, a pickle or a saved cache never keeps the original's addresses: on the host it is refused (its buffers are no
    GPU's), on a GPU they are its own buffers'."""
    cache = BlockCache.__new__(BlockCache)
    for name in ("_kc", "_vc", "_ks", "_vs", "_mean"):
        setattr(cache, name, torch.zeros(2, 1, 64, 64))
    cache.pages, cache.heads, cache.head_dim = 2, 1, 64
    cache.device_index, cache.pointers, cache.mean_pointer = 0, (1, 2, 3, 4), 5
    for again in (copy.deepcopy, copy.copy, lambda c: pickle.loads(pickle.dumps(c))):
        with pytest.raises(ValueError, match="GPU"):
            again(cache)
    torch.save(cache, tmp_path / "cache")
    with pytest.raises(ValueError, match="GPU"):
        torch.load(tmp_path / "cache", weights_only=False)


def _host_rotary(monkeypatch):
    """rotary_axes on the host: the checks and the autograd function as they are, the launch in torch."""
    def turn(q, k, pos, sections, inv_freq, inverse):
        out = []
        for x in (q, k):
            y = None if x is None else torch.from_numpy(O.rotate(x.detach().numpy(), pos.numpy(), sections, inv_freq.detach().numpy(),
                                                                 -1.0 if inverse else 1.0)).to(x.dtype)
            out.append(y)
        return tuple(out)

    monkeypatch.setattr(ops, "_gpu", lambda t, name, dev=-1: 0)
    monkeypatch.setattr(ops, "_rotary", turn)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    g = torch.Generator().manual_seed(0)
    q, k, tq, tk = (torch.randn(2, 3, 5, 8, generator=g) for _ in range(4))
    pos = torch.randint(0, 9, (1, 5, 2), generator=g, dtype=torch.int32).expand(2, 5, 2)
    return turn, q, k, tq, tk, pos, (2, 4), torch.tensor([1.0, 0.5, 0.25], dtype=torch.float64)


def test_rotary_carries_forward_tangents(monkeypatch):
    """A dual tensor's tangent takes the same turn, with and without gradients; an input without one adds zeros."""
    turn, q, k, tq, tk, pos, sections, freq = _host_rotary(monkeypatch)
    want_q, want_k = turn(tq, tk, pos, sections, freq, False)

    def tangents(q, k):
        return [None if x is None else fwd.unpack_dual(x).tangent for x in ops.rotary_axes(q, k, pos, sections, freq)]

    with fwd.dual_level():
        for grad in (False, True):
            a, b = (x.clone().requires_grad_(grad) for x in (q, k))
            got = tangents(fwd.make_dual(a, tq), fwd.make_dual(b, tk))
            assert torch.equal(got[0], want_q) and torch.equal(got[1], want_k)
            got = tangents(a, fwd.make_dual(b, tk))
            assert not got[0].any() and torch.equal(got[1], want_k)
            got = tangents(fwd.make_dual(a, tq), None)
            assert torch.equal(got[0], want_q) and got[1] is None
            with torch.no_grad():
                assert torch.equal(tangents(fwd.make_dual(a, tq), b)[0], want_q)
        t = tq.clone().requires_grad_()  # a derivative of the tangent: the opposite turn
        out = tangents(fwd.make_dual(q, t), k)[0]
        back, = torch.autograd.grad(out, t, tk)
        assert torch.equal(back, turn(tk, None, pos, sections, freq, True)[0])


def test_derivatives_that_are_refused(monkeypatch):
    _, q, k, tq, _, pos, sections, freq = _host_rotary(monkeypatch)
    with pytest.raises(ValueError, match="inv_freq"):
        ops.rotary_axes(q, k, pos, sections, freq.clone().requires_grad_())
    with torch.no_grad():
        ops.rotary_axes(q, k, pos, sections, freq.clone().requires_grad_())
    with fwd.dual_level():
        with pytest.raises(ValueError, match="inv_freq"):
            ops.rotary_axes(q, k, pos, sections, fwd.make_dual(freq, freq))
        for grad in (True, False):  # the block cache has no derivative of either kind
            with torch.set_grad_enabled(grad), pytest.raises(ValueError, match="tangent"):
                ops._inference(fwd.make_dual(q, tq), "q")
        ops._inference(q, "q")
        with pytest.raises(ValueError, match="tangent"):
            stream_attention(None, fwd.make_dual(q, tq), None, None, None, None, None, keep=None)
    with pytest.raises(ValueError, match="gradient"):
        ops._inference(q.requires_grad_(), "q")


def test_frames_from_positions_over_three_axes():
    """A sparse layer reads the grid from the row and column axes, the last two, whatever the time before them."""
    from vasc_amd.aggregator import grid_positions
    from vasc_amd.attention import _infer_frames
    pos = grid_positions(6, 3, 4, 5, "cpu").reshape(1, 6 * 17, 2)
    time = torch.arange(100, 106).repeat_interleave(17).view(1, -1, 1)
    assert _infer_frames(pos, 6 * 17, 5) == (3, 4, 6, 17)
    assert _infer_frames(torch.cat([time, pos], -1), 6 * 17, 5) == (3, 4, 6, 17)


@pytest.mark.parametrize("view", ["leaf", "transpose", "expand", "unbind"])
def test_captured_call_on_views_of_leaves(monkeypatch, view):
    """What q and k are views of counts, through rotary_axes itself; a leaf of another op's graph is not seen."""
    _, q, k, _, _, pos, sections, freq = _host_rotary(monkeypatch)
    capturing = [False]
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing[0])
    make = dict(leaf=lambda: (q.clone().requires_grad_(),) * 2, transpose=lambda: seen(q.transpose(1, 2), lambda t: t.transpose(1, 2)),
                expand=lambda: seen(q[:1, :1], lambda t: t.expand(2, 3, 5, 8)),
                unbind=lambda: seen(torch.stack([q, k]), lambda t: t.view(2, 6, 5, 8).unbind(0)[0].view(2, 3, 5, 8)))

    def seen(t, how):
        leaf = t.clone().requires_grad_()
        return leaf, lambda: how(leaf)

    leaf, call = make[view]()
    of = call if callable(call) else lambda: leaf
    other = k.clone().requires_grad_()
    for args in ((lambda: (of(), None)), (lambda: (other, of())), (lambda: (k, of()))):
        capturing[0] = False
        eager = ops.rotary_axes(*args(), pos, sections, freq)
        capturing[0] = True
        with pytest.raises(ValueError, match="eager graph"):
            ops.rotary_axes(*args(), pos, sections, freq)
        ops.rotary_axes(q.clone().requires_grad_(), None, pos, sections, freq)
        del eager
        ops.rotary_axes(*args(), pos, sections, freq)
    capturing[0] = False
    eager = ops.rotary_axes(leaf * 1 if view == "leaf" else of() * 1, None, pos, sections, freq)
    capturing[0] = True
    ops.rotary_axes(of(), None, pos, sections, freq)
    del eager


def test_rows_of_size_one_dimensions(monkeypatch):
    """The stride of a dimension of size one says nothing: such rows are taken, wherever they start."""
    for x in (torch.zeros(1, 1, 1, 65)[..., :64], torch.zeros(1, 2, 3, 65)[:, 1:2, 2:3, 1:], torch.zeros(1, 3, 1, 64 + 8)[..., 3:67],
              torch.zeros(2, 1, 4, 65)[..., :64], torch.zeros(7, 1, 1, 130)[:, :, :, 1:129]):
        t, ptr, sb, sh, st = ops._rows8(x, "q", (torch.float32,))
        assert t.shape == x.shape and ptr == t.data_ptr() and ptr % 16 == 0 and not (sb | sh | st) % 8
        want = torch.empty(0).set_(t.untyped_storage(), t.storage_offset(), x.shape, (sb, sh, st, 1))
        assert torch.equal(want, x)
    with pytest.raises(ValueError, match="multiple of 8"):
        ops._rows8(torch.zeros(1, 2, 3, 60), "q", (torch.float32,))


def _host_cache(monkeypatch):
    """The cache operators' checks on the host: a cache of 2 heads of 64, and the launches that would have been made."""
    launches = []
    monkeypatch.setattr(ops, "_gpu", lambda t, name, dev=-1: -1)
    monkeypatch.setattr(ops, "_launch", lambda dev, name, *args: launches.append((name, args)))
    return types.SimpleNamespace(heads=2, head_dim=64, device_index=-1, pages=4, pointers=(FAKE,) * 4, mean_pointer=FAKE), launches


def test_out_that_overlaps_itself_or_needs_a_gradient(monkeypatch):
    cache, launches = _host_cache(monkeypatch)
    q, table, n = torch.zeros(2, 4, 3, 64, dtype=torch.bfloat16), torch.zeros(2, 4, dtype=torch.int32), torch.ones(2, dtype=torch.int32)
    one = torch.zeros(1, 1, 1, 64, dtype=torch.bfloat16)
    for out in (one.expand(2, 4, 3, 64), torch.zeros(2, 1, 3, 64, dtype=torch.bfloat16).expand(2, 4, 3, 64)):
        with pytest.raises(ValueError, match="overlap"):
            ops.cache_attn(q, cache, table, n, out=out)
    with pytest.raises(ValueError, match="gradient"):
        ops.cache_attn(q, cache, table, n, out=torch.zeros_like(q).requires_grad_())
    assert not launches
    with torch.no_grad():
        ops.cache_attn(q, cache, table, n, out=torch.zeros_like(q).requires_grad_())
    ops.cache_attn(q[:1, :2, :1], cache, table[:1], n[:1], out=one.expand(1, 2, 1, 64)[:, :1].expand(1, 2, 1, 64).clone())
    assert len(launches) == 2


def test_out_of_size_one_dimensions(monkeypatch):
    """An out whose dimensions of size one have odd strides is taken, with strides that the kernel accepts."""
    cache, launches = _host_cache(monkeypatch)
    table, n = torch.zeros(1, 4, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    q = torch.zeros(1, 2, 1, 64, dtype=torch.bfloat16)
    wide = torch.zeros(1, 2, 3, 68, dtype=torch.bfloat16)
    for out in (torch.zeros(1, 2, 64, 1, dtype=torch.bfloat16).transpose(2, 3).contiguous(), wide[:, :, 1:2, :64],
                torch.zeros(129, dtype=torch.bfloat16)[:128].as_strided((1, 2, 1, 64), (129, 64, 65, 1))):
        assert ops.cache_attn(q, cache, table, n, out=out) is out
        strides = launches[-1][1][5:8]
        assert launches[-1][1][4] == out.data_ptr() and not any(st % 4 for st in strides) and strides[1] == out.stride(1)
    with pytest.raises(ValueError, match="aligned rows"):
        ops.cache_attn(q, cache, table, n, out=torch.zeros(200, dtype=torch.bfloat16).as_strided((1, 2, 1, 64), (128, 65, 64, 1)))


def test_integers_past_32_bits(monkeypatch):
    """Lengths, starts, page tables and lists of 64 bits keep their sense: what is out of range stays out of range."""
    cache, launches = _host_cache(monkeypatch)
    far = torch.tensor([2 ** 32 + 5, -2 ** 32 + 5, 2 ** 31, -2 ** 31 - 1, 2 ** 63 - 1, -2 ** 63, 7, -1])
    got = ops._int_rows(far, "start", 8, -1)
    most = 2 ** 31 - 1
    assert got.dtype == torch.int32 and got.tolist() == [most, -1, most, -1, most, -1, 7, -1]
    assert ops._int_rows(far[6:].to(torch.int8), "start", 2, -1).tolist() == [7, -1]
    table, stride, pages = ops._page_table(far.view(2, 4), 2, -1)
    assert table.dtype == torch.int32 and (stride, pages) == (4, 4) and table.flatten().tolist() == got.tolist()
    q = torch.zeros(1, 2, 1, 64, dtype=torch.bfloat16)
    seen = []
    monkeypatch.setattr(ops, "_ptr", lambda t: seen.append(t))
    ops.cache_attn(q, cache, table[:1], got[6:7], far.view(1, 1, 1, 8).expand(1, 2, 1, 8), far[:1].view(1, 1, 1).expand(1, 2, 1))
    lists = [t for t in seen if t is not None and t.dim() > 2]
    assert lists[0][0, 0, 0].tolist() == got.tolist() and lists[1].flatten().tolist() == [most] * 2
    for bad in (torch.zeros(8), torch.zeros(8, dtype=torch.bool), torch.zeros(8, dtype=torch.complex64)):
        with pytest.raises(ValueError, match="integers"):
            ops._int_rows(bad, "start", 8, -1)


def test_frequencies_made_in_inference_mode_or_loaded_elsewhere(tmp_path):
    """A rope first called in inference mode is trained with later, and one that was saved is loaded for another device."""
    from vasc_amd.aggregator import RotaryPositionEmbeddingAxes
    rope = RotaryPositionEmbeddingAxes((4, 8), 100.0)
    with torch.inference_mode():
        first = rope.frequencies("cpu")
    assert not first.is_inference() and rope.frequencies("cpu") is first
    torch.save(rope, tmp_path / "rope")
    other = torch.load(tmp_path / "rope", map_location="meta", weights_only=False)
    for again in (other, copy.deepcopy(rope), pickle.loads(pickle.dumps(rope))):
        assert again.frequencies("cpu").device.type == "cpu" and torch.equal(again.frequencies("cpu"), first)


def test_layers_run_on_their_tensors_device(monkeypatch):
    """The layout kernels launch on the current device's stream: a layer whose tokens are on another one makes that current."""
    current, seen = [0], []

    class Device:
        def __init__(self, dev):
            self.dev = dev if isinstance(dev, int) else dev.index

        def __enter__(self):
            self.before, current[0] = current[0], self.dev

        def __exit__(self, *_):
            current[0] = self.before

    def stop(*_):
        seen.append(current[0])
        raise KeyError("stopped")

    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: current[0])
    where = {"x": 3, "pos": 3, "images": 3}
    monkeypatch.setattr(ops, "_gpu", lambda t, name, dev=-1: where[name])
    attn = types.SimpleNamespace(num_heads=2, qkv=stop)
    x = torch.zeros(1, 4, 128)
    with pytest.raises(KeyError):
        stream_attention(attn, x, torch.zeros(1, 4, 2), None, None, None, None, keep=None)
    model = types.SimpleNamespace(_resnet_mean=0, _resnet_std=1, patch_embed=types.SimpleNamespace(
        weight=x, bias=None, kernel_size=(2, 2), stride=(1, 1), padding=0, __call__=stop))
    model.patch_embed = type("Conv", (), dict(vars(model.patch_embed), __call__=lambda self, x: stop()))()
    with pytest.raises(KeyError):
        AggregatorStream(model, 4).push(torch.zeros(1, 1, 3, 4, 4))
    assert seen == [3, 3] and current == [0]


def test_streamed_layer_refuses_tensors_elsewhere():
    x = torch.zeros(1, 4, 128)
    with pytest.raises(ValueError, match="x must be a GPU"):
        stream_attention(None, x, None, None, None, None, None, keep=None)
    with pytest.raises(ValueError, match="images must be a GPU"):
        AggregatorStream(None, 4).push(torch.zeros(1, 1, 3, 4, 4))
