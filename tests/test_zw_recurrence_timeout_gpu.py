"""The error path of the linear recurrence's waits: one that is given up ends, is counted, and leaves NaN where the
missing map went in and nowhere else.  (Runs behind the tests that ask that no wait was given up in the process.)"""
import ctypes
import os

import pytest
import torch

import gpu_util
import thrust_amd
from conftest import EMULATED
from lm_util import get, put
from thrust_amd import capi

pytestmark = pytest.mark.gpu

# workgroups run one after the other in an emulated session unless it asks for more: then nothing is ever waited for
WAITS = not EMULATED or os.environ.get("THRUST_CDNA4_EMULATED_RESIDENT", "1").partition(":")[0] != "1"


def counted():
    """Both ways to the count."""
    gpu_util.synchronize()
    c, where = ctypes.c_ulonglong(0), ctypes.c_void_p()
    capi.check(capi.lib().thrust_cdna4_lookback_timeouts(ctypes.byref(c)), "lookback_timeouts")
    capi.check(capi.lib().thrust_cdna4_lookback_timeout_counter(ctypes.byref(where)), "lookback_timeout_counter")
    word = ctypes.c_uint32(0)
    capi.check(capi.lib().thrust_cdna4_read_back(ctypes.byref(word), where, 4, gpu_util.stream_handle()), "read_back")
    assert word.value == c.value & 0xffffffff
    return c.value


@pytest.mark.parametrize("channels", [3, 140])
def test_a_wait_that_is_given_up(channels):
    L = capi.lib()
    rows, batch = 2000, 3
    g = torch.Generator().manual_seed(channels)
    shape = (batch, rows, channels)
    gate, x, grad_out = (torch.rand(shape, generator=g), torch.randn(shape, generator=g), torch.randn(shape, generator=g))
    init, grad_final = torch.randn((batch, channels), generator=g), torch.randn((batch, channels), generator=g)
    d = [put(t) for t in (gate, x, init, grad_out, grad_final)]

    def one():
        out, final, states = thrust_amd.linear_scan(d[0], d[1], init=d[2], return_states=True)
        return get(out), get(final), states

    def back(states):
        return [get(t) for t in thrust_amd.linear_scan_backward(d[3], d[0], d[1], states, init=d[2], grad_final=d[4])]
    out, final, states = one()
    grads = back(states)
    before = counted()
    prev_limit = L.thrust_cdna4_set_test_sort_spin_limit(0)
    prev_delay = L.thrust_cdna4_set_test_publish_delay(200)
    try:
        got, got_final, _ = one()
        between = counted()
        got_grads = back(states)
    finally:
        L.thrust_cdna4_set_test_publish_delay(prev_delay)
        L.thrust_cdna4_set_test_sort_spin_limit(prev_limit)
    after = counted()
    for a, b in zip([got, got_final] + got_grads, [out, final] + grads):
        assert (torch.isnan(a) | (a == b)).all()
    # the first tile in either direction waits for nothing
    assert torch.equal(got[:, :64], out[:, :64]) and torch.equal(got_grads[1][:, -(rows % 64):], grads[1][:, -(rows % 64):])
    if WAITS:
        assert before < between < after
        # each chain's last tile needs the first one's map, which was late
        assert torch.isnan(got_final).all() and torch.isnan(got_grads[2]).all()
    else:
        assert before == between == after
    again, again_final, _ = one()
    assert torch.equal(again, out) and torch.equal(again_final, final) and all(torch.equal(a, b) for a, b in zip(back(states), grads))
    assert counted() == after


def test_a_sequence_that_needs_no_missing_map_is_whole():
    """Packed: tile 0 is late, and only the sequence that comes out of it can miss it."""
    L = capi.lib()
    lengths = [30, 400, 60, 50]  # the second one leaves tile 0; the last two lie in other tiles, each in one
    offsets = torch.tensor([0] + lengths).cumsum(0).int()
    g = torch.Generator().manual_seed(1)
    gate, x = torch.rand((540, 5), generator=g), torch.randn((540, 5), generator=g)
    d = [put(t) for t in (gate, x, offsets)]
    out, final = (get(t) for t in thrust_amd.linear_scan(d[0], d[1], offsets=d[2]))
    prev_limit = L.thrust_cdna4_set_test_sort_spin_limit(0)
    prev_delay = L.thrust_cdna4_set_test_publish_delay(200)
    try:
        got, got_final = (get(t) for t in thrust_amd.linear_scan(d[0], d[1], offsets=d[2]))
    finally:
        L.thrust_cdna4_set_test_publish_delay(prev_delay)
        L.thrust_cdna4_set_test_sort_spin_limit(prev_limit)
    assert torch.equal(got[:64], out[:64]) and torch.equal(got[430:448], out[430:448]) and torch.equal(got_final[0], final[0])
    assert (torch.isnan(got) | (got == out)).all()
    if WAITS:
        assert torch.isnan(got_final[1]).all()
