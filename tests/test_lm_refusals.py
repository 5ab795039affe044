"""CPU-only: what the entry points of the linear recurrence and the page cache refuse, and their size
queries, which touch no device."""
import contextlib
import ctypes

import pytest
import torch

import thrust_amd
from thrust_amd import capi, device

INVALID = 1


def scan_args(**change):
    a = dict(gate_dtype=capi.F32, x_dtype=capi.BF16, batch=2, rows=1000, channels=300, gate=0x1000, x=0x100000000, out=0x200000000,
             gate_batch_stride=300000, gate_row_stride=300, x_batch_stride=300000, x_row_stride=300, out_batch_stride=300000, out_row_stride=300)
    return capi.LinearScanArgs(**dict(a, **change))


def size(entry, args):
    nb = ctypes.c_size_t(0)
    return entry(None, ctypes.byref(nb), ctypes.byref(args), None), nb.value


def test_size_queries():
    L = capi.lib()
    rc, many = size(L.thrust_cdna4_linear_scan, scan_args())
    assert rc == 0 and 16 * 2 * 300 * 8 <= many < 40 * 2 * 300 * 8  # a map for each channel of 16 tiles
    rc, one = size(L.thrust_cdna4_linear_scan, scan_args(rows=64))
    assert rc == 0 and one == 256  # not touched: a single tile
    assert size(L.thrust_cdna4_linear_scan, scan_args(batch=0))[0] == 0
    for entry in (L.thrust_cdna4_pages_compact,):
        nb = ctypes.c_size_t(0)
        assert entry(None, ctypes.byref(nb), ctypes.byref(cache_args()), None, None, None, None) == 0 and nb.value >= 1000 * 16


@pytest.mark.parametrize("change", [
    dict(gate_dtype=capi.F64), dict(x_dtype=capi.F64, gate_dtype=capi.F64), dict(x_dtype=capi.I32), dict(gate_dtype=capi.F16), dict(x_dtype=99),
    dict(batch=-1), dict(rows=-1), dict(channels=-1), dict(batch=2 ** 31), dict(channels=2 ** 31), dict(channels=2 ** 28 + 1, rows=1), dict(rows=2 ** 50), dict(batch=1, rows=2 ** 31, channels=256),
    dict(offset_bytes=2, batch=1), dict(offset_bytes=4, batch=2), dict(offset_bytes=8, batch=1, sequences=-1), dict(offset_bytes=8, batch=1, sequences=2 ** 31)],
    ids=str)
def test_shapes_and_types_refused(change):
    L = capi.lib()
    assert size(L.thrust_cdna4_linear_scan, scan_args(**change))[0] == INVALID
    fields = {k: getattr(scan_args(**change), k) for k in ("gate_dtype", "x_dtype", "batch", "rows", "channels", "offset_bytes", "sequences")}
    assert size(L.thrust_cdna4_linear_scan_backward, capi.LinearScanBackwardArgs(**fields))[0] == INVALID


@pytest.mark.parametrize("change", [dict(gate=None), dict(x=None), dict(out=None), dict(offset_bytes=4, batch=1, sequences=3),
                                    dict(init=0x5000, final_state=0x5000), dict(init=0x5000, final_state=0x5000 + 4 * 599)], ids=str)
def test_ranges_refused_before_anything_is_launched(change):
    L = capi.lib()
    nb = ctypes.c_size_t(1 << 30)
    assert L.thrust_cdna4_linear_scan(0x10000, ctypes.byref(nb), ctypes.byref(scan_args(**change)), None) == INVALID
    assert L.thrust_cdna4_linear_scan(0x10004, ctypes.byref(nb), ctypes.byref(scan_args()), None) == INVALID  # the storage's alignment
    small = ctypes.c_size_t(255)
    assert L.thrust_cdna4_linear_scan(0x10000, ctypes.byref(small), ctypes.byref(scan_args()), None) == INVALID
    assert L.thrust_cdna4_linear_scan(0x10000, None, ctypes.byref(scan_args()), None) == INVALID
    assert L.thrust_cdna4_linear_scan(0x10000, ctypes.byref(nb), None, None) == INVALID


def test_backward_refuses():
    L = capi.lib()
    nb = ctypes.c_size_t(1 << 30)
    good = dict(gate_dtype=capi.F32, x_dtype=capi.F32, batch=1, rows=10, channels=10, gate=0x10000, x=0x20000, grad_out=0x30000, grad_gate=0x40000,
                grad_x=0x50000, states=0x60000, gate_row_stride=10, x_row_stride=10, grad_out_row_stride=10, grad_gate_row_stride=10, grad_x_row_stride=10)
    for change in (dict(gate=None), dict(x=None), dict(grad_out=None), dict(grad_gate=None), dict(grad_x=None), dict(states=None),
                   dict(grad_init=0x7000, grad_final=0x7010), dict(grad_init=0x7000, init=0x7010)):
        args = capi.LinearScanBackwardArgs(**dict(good, **change))
        assert L.thrust_cdna4_linear_scan_backward(0x10000, ctypes.byref(nb), ctypes.byref(args), None) == INVALID, change


def test_step_refuses():
    call = capi.lib().thrust_cdna4_linear_scan_step

    def rc(gate_dtype=capi.F32, x_dtype=capi.F32, gate=0x1000, x=0x2000, out=0x3000, state=0x4000, slots_n=8, slots=None, batch=4, channels=4):
        return call(gate_dtype, x_dtype, 0, gate, 4, x, 4, out, 4, state, slots_n, slots, batch, channels, None)
    assert rc(batch=0) == 0 and rc(channels=0) == 0
    for bad in (dict(batch=9), dict(batch=-1), dict(channels=-1), dict(slots_n=-1), dict(gate=None), dict(x=None), dict(out=None), dict(state=None),
                dict(gate_dtype=capi.BF16), dict(x_dtype=capi.F64), dict(batch=2 ** 31, slots_n=2 ** 32), dict(channels=2 ** 31), dict(batch=2 ** 24, slots_n=2 ** 24)):
        assert rc(**bad) == INVALID, bad


def cache_args(**change):
    a = dict(pools=0x1000, page_bytes=64, num_pools=2, num_pages=1000, page_size=16, num_sequences=10, max_pages=8, tables=0x2000, lengths=0x3000, refs=0x4000)
    return capi.PageCacheArgs(**dict(a, **change))


def test_page_calls_refuse():
    L = capi.lib()
    nb = ctypes.c_size_t(1 << 30)
    t, b = 0x10000, ctypes.byref(nb)

    def calls(cache, temp=t, ids=0x5000, done=0x6000, n=3):
        c = ctypes.byref(cache)
        return {L.thrust_cdna4_pages_fork(temp, b, c, ids, ids, n, 1, done, None), L.thrust_cdna4_pages_resize(temp, b, c, ids, ids, n, done, None)}
    for bad in (dict(num_pools=-1), dict(num_pages=-1), dict(page_bytes=-1), dict(page_size=0), dict(num_sequences=-1), dict(max_pages=-1),
                dict(page_size=1 << 20, max_pages=1 << 11), dict(pools=None), dict(tables=None), dict(lengths=None), dict(refs=None)):
        assert calls(cache_args(**bad)) == {INVALID}, bad
        assert L.thrust_cdna4_pages_free(ctypes.byref(cache_args(**bad)), 0x5000, 3, None, None) == INVALID, bad
        assert L.thrust_cdna4_pages_compact(t, b, ctypes.byref(cache_args(**bad)), 0x5000, 0x6000, 0x7000, None) == INVALID, bad
    assert calls(cache_args(), temp=0x10004) == {INVALID} and calls(cache_args(), ids=None) == {INVALID} and calls(cache_args(), done=None) == {INVALID}
    assert calls(cache_args(), n=-1) == {INVALID} and calls(cache_args(), n=(1 << 23) + 1) == {INVALID} and calls(cache_args(), n=0) == {0}
    small = ctypes.c_size_t(100)
    assert L.thrust_cdna4_pages_fork(t, ctypes.byref(small), ctypes.byref(cache_args()), 0x5000, 0x5000, 3, 1, 0x6000, None) == INVALID
    assert L.thrust_cdna4_pages_free(None, 0x5000, 3, None, None) == INVALID and L.thrust_cdna4_pages_free(ctypes.byref(cache_args()), 0x5000, 0, None, None) == 0
    for out in ((None, 0x6000, 0x7000), (0x5000, None, 0x7000), (0x5000, 0x6000, None)):
        assert L.thrust_cdna4_pages_compact(t, b, ctypes.byref(cache_args()), *out, None) == INVALID


def test_other_entry_points_refuse_16_bit_types():
    L = capi.lib()
    for code in (capi.F16, capi.BF16):
        nb = ctypes.c_size_t(0)
        assert L.thrust_cdna4_scan(None, ctypes.byref(nb), code, capi.PLUS, 0, None, None, 5, None, None) == INVALID
        assert L.thrust_cdna4_sort_keys(None, ctypes.byref(nb), code, None, 5, 0, None) == INVALID
        assert L.thrust_cdna4_scan_by_key(None, ctypes.byref(nb), capi.I32, code, capi.PLUS, 0, None, None, None, 5, None, None) == INVALID
        assert L.thrust_cdna4_histogram_even(None, ctypes.byref(nb), code, None, 5, None, 4, 0.0, 1.0, None) == INVALID


# ---------------------------------------------------------------------------------------
# The Python layer
# ---------------------------------------------------------------------------------------
def test_no_cpu_path():
    x = torch.zeros(1, 2, 3)
    with pytest.raises(ValueError, match="device tensors"):
        thrust_amd.linear_scan(x, x)
    with pytest.raises(ValueError, match="device tensors"):
        thrust_amd.linear_scan_step(x[0], x[0], x[0])
    with pytest.raises(ValueError, match="device tensors"):
        thrust_amd.PageCache([x], 4, 1, 1)


@pytest.fixture
def any_device(monkeypatch):
    """The checks that come after the device's, on host tensors: nothing may be launched."""
    monkeypatch.setattr(device, "need_device", lambda *t: torch.device("cpu"))
    monkeypatch.setattr(device, "current", lambda d: pytest.fail("not refused"))
    monkeypatch.setattr(device, "is_current", lambda d: pytest.fail("not refused"))
    monkeypatch.setattr(device, "stream", lambda d: 0)


Z = torch.zeros
SCANS = {
    "types": lambda: thrust_amd.linear_scan(Z(1, 2, 3).half(), Z(1, 2, 3)),
    "64 bits": lambda: thrust_amd.linear_scan(Z(1, 2, 3).double(), Z(1, 2, 3).double()),
    "shapes": lambda: thrust_amd.linear_scan(Z(1, 2, 3), Z(1, 2, 4)),
    "broadcast": lambda: thrust_amd.linear_scan(Z(1, 2, 1), Z(1, 2, 4)),
    "two dimensions": lambda: thrust_amd.linear_scan(Z(2, 3), Z(2, 3)),
    "three dimensions, packed": lambda: thrust_amd.linear_scan(Z(1, 2, 3), Z(1, 2, 3), offsets=Z(2).int()),
    "offsets of floats": lambda: thrust_amd.linear_scan(Z(2, 3), Z(2, 3), offsets=Z(2)),
    "no offsets": lambda: thrust_amd.linear_scan(Z(2, 3), Z(2, 3), offsets=Z(0).int()),
    "offsets apart": lambda: thrust_amd.linear_scan(Z(2, 3), Z(2, 3), offsets=Z(4).int()[::2]),
    "channels apart": lambda: thrust_amd.linear_scan(Z(1, 2, 3), Z(1, 2, 6)[..., ::2]),
    "init's shape": lambda: thrust_amd.linear_scan(Z(1, 2, 3), Z(1, 2, 3), init=Z(2, 3)),
    "init's type": lambda: thrust_amd.linear_scan(Z(1, 2, 3), Z(1, 2, 3), init=Z(1, 3).half()),
    "out's type": lambda: thrust_amd.linear_scan(Z(1, 2, 3), Z(1, 2, 3), out=Z(1, 2, 3).half()),
    "out's shape": lambda: thrust_amd.linear_scan(Z(1, 2, 3), Z(1, 2, 3), out=Z(1, 3, 3)),
    "out expanded": lambda: thrust_amd.linear_scan(Z(2, 2, 3), Z(2, 2, 3), out=Z(1, 2, 3).expand(2, 2, 3)),
    "out's rows overlap": lambda: thrust_amd.linear_scan(Z(1, 2, 3), Z(1, 2, 3), out=Z(9).as_strided((1, 2, 3), (9, 2, 1))),
    "wants its gradient": lambda: thrust_amd.linear_scan(Z(1, 2, 3), Z(1, 2, 3).requires_grad_()),
    "states' shape": lambda: thrust_amd.linear_scan_backward(Z(1, 65, 3), Z(1, 65, 3), Z(1, 65, 3), Z(1, 1, 3)),
    "states' type": lambda: thrust_amd.linear_scan_backward(Z(1, 5, 3), Z(1, 5, 3), Z(1, 5, 3), Z(1, 1, 3).half()),
    "grad_out's type": lambda: thrust_amd.linear_scan_backward(Z(1, 5, 3).half(), Z(1, 5, 3), Z(1, 5, 3), Z(1, 1, 3)),
    "grad_out's shape": lambda: thrust_amd.linear_scan_backward(Z(1, 4, 3), Z(1, 5, 3), Z(1, 5, 3), Z(1, 1, 3)),
    "grad_final's shape": lambda: thrust_amd.linear_scan_backward(Z(1, 5, 3), Z(1, 5, 3), Z(1, 5, 3), Z(1, 1, 3), grad_final=Z(3)),
    "step: three dimensions": lambda: thrust_amd.linear_scan_step(Z(1, 2, 3), Z(1, 2, 3), Z(2, 3)),
    "step: state's type": lambda: thrust_amd.linear_scan_step(Z(2, 3), Z(2, 3), Z(2, 3).half()),
    "step: state's width": lambda: thrust_amd.linear_scan_step(Z(2, 3), Z(2, 3), Z(2, 4)),
    "step: slots' type": lambda: thrust_amd.linear_scan_step(Z(2, 3), Z(2, 3), Z(2, 3), slots=Z(2).long()),
    "step: slots' number": lambda: thrust_amd.linear_scan_step(Z(2, 3), Z(2, 3), Z(2, 3), slots=Z(3).int()),
    "step: too few slots": lambda: thrust_amd.linear_scan_step(Z(2, 3), Z(2, 3), Z(1, 3)),
    "step: out's type": lambda: thrust_amd.linear_scan_step(Z(2, 3), Z(2, 3), Z(2, 3), out=Z(2, 3).half()),
    "cache: no pool": lambda: thrust_amd.PageCache([], 4, 1, 1),
    "cache: pages differ": lambda: thrust_amd.PageCache([Z(3, 2), Z(4, 2)], 4, 1, 1),
    "cache: bytes differ": lambda: thrust_amd.PageCache([Z(3, 2), Z(3, 2).half()], 4, 1, 1),
    "cache: pages apart": lambda: thrust_amd.PageCache([Z(6, 2)[::2]], 4, 1, 1),
    "cache: page size": lambda: thrust_amd.PageCache([Z(3, 2)], 0, 1, 1),
    "cache: lengths past 2^31": lambda: thrust_amd.PageCache([Z(3, 2)], 1 << 20, 1, 1 << 11),
    "cache: tables' shape": lambda: thrust_amd.PageCache([Z(3, 2)], 4, 2, 2, tables=Z(2, 3).int()),
    "cache: refs' type": lambda: thrust_amd.PageCache([Z(3, 2)], 4, 2, 2, refs=Z(3)),
    "resize: lengths' type": lambda: thrust_amd.PageCache([Z(3, 2)], 4, 2, 2).resize(Z(2).int(), Z(2).long()),
    "resize: numbers differ": lambda: thrust_amd.PageCache([Z(3, 2)], 4, 2, 2).resize(Z(2).int(), Z(3).int()),
    "fork: apart": lambda: thrust_amd.PageCache([Z(3, 2)], 4, 2, 2).fork(Z(4).int()[::2], Z(2).int()),
    "compact: one of two": lambda: thrust_amd.PageCache([Z(3, 2)], 4, 2, 2).compact(refs=Z(3).int()),
    "compact: shape": lambda: thrust_amd.PageCache([Z(3, 2)], 4, 2, 2).compact(tables=Z(2, 2).int(), refs=Z(4).int()),
}


@pytest.mark.parametrize("what", list(SCANS), ids=str)
def test_refused_with_a_value_error(any_device, what):
    # (a cache's own check of requests compares devices, which are host ones here)
    with pytest.raises(ValueError):
        SCANS[what]()


def test_a_forward_gradient_is_not_dropped(any_device):
    """A dual tensor does not want a gradient of its own, and its tangent would be lost."""
    from torch.autograd import forward_ad
    x, state = Z(1, 5, 3), Z(5, 3)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        flat, two = forward_ad.make_dual(Z(5, 3), torch.ones(5, 3)), forward_ad.make_dual(Z(1, 3), torch.ones(1, 3))
        for call in (lambda: thrust_amd.linear_scan(dual, x), lambda: thrust_amd.linear_scan(x, dual), lambda: thrust_amd.linear_scan(x, x, init=two),
                     lambda: thrust_amd.linear_scan(x, x, out=dual),
                     lambda: thrust_amd.linear_scan_backward(dual, x, x, Z(1, 1, 3)), lambda: thrust_amd.linear_scan_backward(x, x, x, Z(1, 1, 3), grad_final=two),
                     lambda: thrust_amd.linear_scan_step(flat, state, Z(5, 3)), lambda: thrust_amd.linear_scan_step(state, state, flat)):
            for mode in (torch.enable_grad, torch.no_grad):  # which says nothing of forward mode
                with mode(), pytest.raises(ValueError, match="differentiation"):
                    call()


def test_an_output_that_wants_its_gradient_is_refused(any_device):
    x = Z(1, 5, 3)
    with pytest.raises(ValueError, match="differentiation"):
        thrust_amd.linear_scan(x, x, out=Z(1, 5, 3).requires_grad_())
    with pytest.raises(ValueError, match="differentiation"):
        thrust_amd.linear_scan_step(x[0], x[0], Z(5, 3), out=Z(5, 3).requires_grad_())


class Handle:
    """Stands for the tensor of a cache's pool addresses."""

    def __init__(self):
        self.recorded = []

    def record_stream(self, stream):
        self.recorded.append(stream)


def test_what_a_call_reads_outlives_it(monkeypatch):
    """Private memory that pending work reads is recorded on every stream but its own, once, and kept for good where a graph has it."""
    now = {"stream": 5, "capturing": False}
    monkeypatch.setattr(device, "stream", lambda d: now["stream"])
    monkeypatch.setattr(device, "capturing", lambda: now["capturing"])
    monkeypatch.setattr(torch.cuda, "current_stream", lambda d=None: now["stream"])
    monkeypatch.setattr(device, "_CAPTURED", [])
    on = torch.device("cuda", 0)
    for own in (5, 0):
        now.update(stream=own, capturing=False)
        handle = Handle()
        kept = device.Outliving(handle, on)
        kept.used(own)
        assert handle.recorded == []
        for s, want in ((9, [9]), (9, [9]), (own, [9]), (11, [9, 11])):
            now["stream"] = s
            kept.used(s)
            assert handle.recorded == want
        now.update(stream=12, capturing=True)
        kept.used(12)
        kept.used(12)
        assert handle.recorded == [9, 11] and device._CAPTURED[-1] is handle and device._CAPTURED.count(handle) == 1
        now["capturing"] = False
        kept.used(12)
        assert handle.recorded == [9, 11, 12]


def test_the_calls_that_copy_pages_hold_the_pools_addresses(monkeypatch):
    class Entry:
        def __getattr__(self, name):
            return lambda *a: 0
    monkeypatch.setattr(device, "need_device", lambda *t: torch.device("cpu"))
    monkeypatch.setattr(device, "stream", lambda d: 0)
    monkeypatch.setattr(device, "is_current", lambda d: True)
    monkeypatch.setattr(capi, "lib", Entry)
    monkeypatch.setattr(device, "stream", lambda d: 3)
    cache = thrust_amd.PageCache([Z(3, 2)], 4, 2, 2)
    uses = []
    monkeypatch.setattr(type(cache._pointers), "used", lambda self, stream: uses.append(self))
    cache.resize(Z(1).int(), Z(1).int())
    cache.fork(Z(1).int(), Z(1).int())
    cache.compact()
    assert uses == [cache._pointers] * 3
    monkeypatch.setattr(device, "stream", lambda d: 0)  # back on the default one, which is not where it was made
    cache.compact()
    assert uses == [cache._pointers] * 4


# `out` may be x or gate; every other overlap of an output with an input would be written while it is read
OVERLAPS = {  # of a buffer [9, 2, 12]
    "shifted by a row": lambda b: (b[1:7, 0, :4][None], b[0:6, 0, :4][None]),
    "shifted by a column": lambda b: (b[0:6, 0, 1:5][None], b[0:6, 0, 0:4][None]),
    "at another pitch": lambda b: (b.flatten()[:24].view(1, 6, 4), b.flatten()[8:80].view(1, 6, 12)[..., :4]),
    "batches for rows": lambda b: (b[0:2, :, :4], b.as_strided((2, 2, 4), (12, 24, 1))),
    "a row of it": lambda b: (b[0:6, 0, :4][None], b[3:4, 0, :4].expand(6, 4)[None]),
}


@pytest.mark.parametrize("which", list(OVERLAPS), ids=str)
def test_an_output_that_meets_an_input_is_refused(any_device, which):
    out, other = OVERLAPS[which](Z(9, 2, 12))
    fresh = torch.zeros(out.shape)
    for gate, x in ((other, fresh), (fresh, other)):
        with pytest.raises(ValueError, match="shares memory"):
            thrust_amd.linear_scan(gate, x, out=out)
        if len(out) == 1:
            with pytest.raises(ValueError, match="shares memory"):
                thrust_amd.linear_scan_step(gate[0], x[0], Z(8, 4), out=out[0])
    state = Z(8, 4)
    with pytest.raises(ValueError, match="shares memory"):
        thrust_amd.linear_scan_step(fresh[0], fresh[0], state, out=state[1:1 + fresh.shape[1]])
    rows = Z(3, 4)
    with pytest.raises(ValueError, match="shares memory"):
        thrust_amd.linear_scan(Z(1, 3, 4), Z(1, 3, 4), init=rows[1:2], out=rows[None])


def test_a_state_that_meets_what_a_step_reads_or_writes_is_refused(any_device, monkeypatch):
    monkeypatch.setattr(device, "is_current", lambda d: True)  # it is the entry point that refuses, before anything is launched
    rows = Z(8, 12)
    state, x = rows.flatten()[:32].view(8, 4), Z(3, 4)
    for other in (state[2:5], rows[2:5, 4:8], rows[0:1, 8:].expand(3, 4), rows.view(torch.int32).view(torch.float32)[1:4, :4]):
        for gate, v in ((other, x), (x, other)):
            with pytest.raises(ValueError, match="shares memory"):
                thrust_amd.linear_scan_step(gate, v, state)
    call = capi.lib().thrust_cdna4_linear_scan_step

    def meets(at, pitch, batch=5, channels=4, slots=8, state=0x100000):
        return call(capi.F32, capi.F32, 0, 0x1000, 4, at, pitch, 0x4000, 4, state, slots, None, batch, channels, None)
    for at, pitch in ((0x100000, 4), (0x100000 - 16 * 4, 4), (0x100000 - 15, 0), (0x100000 - 4 * 4 * 1000 - 15, 1000), (0x100000 + 127, 1000)):
        assert meets(at, pitch) == INVALID, (hex(at), pitch)


def test_whether_views_share_an_element():
    """Against the sets of addresses, over random views of one buffer."""
    from thrust_amd import recurrence
    g = torch.Generator().manual_seed(2)

    def pick(low, high):
        return int(torch.randint(low, high + 1, (1,), generator=g))

    def addresses(t):
        at = [t.data_ptr()]
        for n, s in zip(t.shape, t.stride()):
            at = [a + k * s * t.element_size() for a in at for k in range(n)]
        return {a + k for a in at for k in range(t.element_size())}
    met = 0
    for _ in range(3000):
        buffer = torch.zeros(400)
        views = []
        for _ in range(2):
            c, n, b = pick(1, 5), pick(1, 5), pick(1, 3)
            rs = pick(0 if views else c, 12)
            bs = pick(0, 40) if views else rs * n + pick(0, 8)
            if views and pick(0, 1):
                (c, n, b), (bs, rs) = views[0].shape[::-1], views[0].stride()[:2]
            v = buffer if pick(0, 3) else buffer.view(torch.bfloat16)
            views.append(v.as_strided((b, n, c), (bs, rs, 1), pick(0, 150)))
        out, t = views
        want = bool(addresses(out) & addresses(t))
        met += want
        assert recurrence._meet(out, t) == want, (out.shape, out.stride(), out.storage_offset(), t.shape, t.stride(), t.storage_offset())
    assert 500 < met < 2500
    assert not recurrence._meet(torch.zeros(0, 3), buffer) and not recurrence._meet(buffer[:0].view(0, 2, 3), buffer)
    big = torch.zeros(1, 8).expand(1 << 40, 8)  # a row that is read again and again is one
    assert recurrence._meet(big[:1, :3], big)


@pytest.mark.parametrize("what", ["tables", "lengths", "refs"])
def test_a_caches_arrays_are_not_replaced(any_device, what):
    """The calls go on with the arrays that the cache was made with: another one in their place would be passed over."""
    cache = thrust_amd.PageCache([Z(3, 2)], 4, 2, 2)
    was = getattr(cache, what)
    with pytest.raises(AttributeError):
        setattr(cache, what, was.clone())
    assert getattr(cache, what) is was


def test_compact_refuses_outputs_that_meet_the_caches_arrays(any_device, monkeypatch):
    monkeypatch.setattr(device, "current", lambda d: contextlib.nullcontext())  # it is the entry point that refuses, before anything is launched
    rows, counts = torch.full((5, 2), -1, dtype=torch.int32), Z(9).int()
    cache = thrust_amd.PageCache([Z(3, 2)], 4, 4, 2, tables=rows[:4], refs=counts[:3])
    for tables, refs in ((rows[1:], Z(3).int()), (Z(4, 2).int(), counts[2:5]), (Z(4, 2).int(), rows.flatten()[:3])):
        with pytest.raises(ValueError, match="share memory"):
            cache.compact(tables=tables, refs=refs)


def test_addresses_are_compared_on_the_host():
    """Whatever torch's default device is."""
    from thrust_amd import recurrence
    b = torch.zeros(9, 12)
    with torch.device("meta"):
        assert recurrence._meet(b[1:7, :4], b[0:6, :4]) and not recurrence._meet(b[1:7, :4], b.as_strided((3, 2, 4), (24, 12, 1), 4))
