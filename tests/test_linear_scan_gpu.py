"""The linear recurrence, its gradient and its step on the GPU against their definitions in 64 bits."""
import ctypes

import pytest
import torch

import gpu_util
import thrust_amd
from conftest import EMULATED
from lm_util import Recurrence, check, get, put
from thrust_amd import capi

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TYPES = [(F32, F32), (F16, F16), (BF16, BF16), (F32, F16), (F32, BF16)]  # gate, x


def name(t):
    return str(t).replace("torch.", "")


def inputs(seed, shape, sequences, gate, x, log):
    g = torch.Generator().manual_seed(seed)
    keep = -torch.exp(torch.empty(shape).uniform_(-6, 0.7, generator=g))  # log of the gate
    sign = torch.where(torch.rand(shape, generator=g) < 0.1, -1.0, 1.0)
    return ((keep if log else keep.exp() * sign).to(gate), torch.randn(shape, generator=g).to(x),
            torch.randn((sequences, shape[-1]), generator=g), torch.randn(shape, generator=g).to(x), torch.randn((sequences, shape[-1]), generator=g))


def offsets_of(lengths, first=0):
    return torch.tensor([first] + lengths).cumsum(0)


def forward(gate, x, init, offsets, log, **more):
    return thrust_amd.linear_scan(put(gate), put(x), init=put(init), offsets=put(offsets), log_gate=log, **more)


def both_ways(seed, shape, gate_t, x_t, log, offsets=None, with_init=True, with_final=True):
    sequences = shape[0] if offsets is None else offsets.numel() - 1
    gate, x, init, grad_out, grad_final = inputs(seed, shape, sequences, gate_t, x_t, log)
    init, grad_final = init if with_init else None, grad_final if with_final else None
    ref = Recurrence(gate, x, init, offsets, log).gradient(grad_out, grad_final)
    d = [put(t) for t in (gate, x, init, offsets, grad_out, grad_final)]
    out, final, states = thrust_amd.linear_scan(d[0], d[1], init=d[2], offsets=d[3], log_gate=log, return_states=True)
    assert out.dtype == x_t and final.dtype == F32 and states.dtype == F32
    check(get(out), ref.out, ref.error_out, "out")  # rows outside every sequence: zero
    check(get(final), ref.final, ref.error_final, "final")
    for b in range(ref.shape[0]):
        for k, t in enumerate(range(0, ref.shape[1], 64)):
            if ref.inside[b, t]:
                check(get(states)[b, k], ref.before[b, t], ref.error_before[b, t], "states")
    grad_gate, grad_x, grad_init = thrust_amd.linear_scan_backward(d[4], d[0], d[1], states, init=d[2], grad_final=d[5], offsets=d[3], log_gate=log)
    assert grad_gate.dtype == gate_t and grad_x.dtype == x_t
    check(get(grad_x), ref.grad_x, ref.error_x, "grad_x")
    check(get(grad_gate), ref.grad_gate, ref.error_gate, "grad_gate")
    if with_init:
        check(get(grad_init), ref.grad_init, ref.error_init, "grad_init")
    else:
        assert grad_init is None


SHAPES = [(1, 1, 1), (2, 1, 5), (3, 7, 3), (1, 63, 64), (2, 64, 65), (1, 65, 129), (1, 127, 133), (2, 129, 132), (1, 200, 261), (5, 16, 6)]


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("gate_t,x_t", TYPES, ids=name)
def test_dense(shape, gate_t, x_t):
    both_ways(sum(shape), shape, gate_t, x_t, log=(shape[1] + shape[2]) % 2 == 0)


@pytest.mark.parametrize("gate_t,x_t", TYPES, ids=name)
@pytest.mark.parametrize("log", [False, True])
def test_many_tiles(gate_t, x_t, log):
    """Past a group of 8 tiles; and of a narrow layer."""
    both_ways(1, (2, 1300, 2), gate_t, x_t, log)
    both_ways(2, (1, 1100, 130), gate_t, x_t, log)


@pytest.mark.parametrize("gate_t,x_t", [(F32, F32), (BF16, BF16)], ids=name)
def test_past_super_groups(gate_t, x_t):
    both_ways(3, (1, 9000, 1), gate_t, x_t, False)  # 64-row tiles: 141 of them; 128-row tiles: 71
    both_ways(4, (1, 17000, 1), gate_t, x_t, True)


@pytest.mark.parametrize("with_init,with_final", [(False, True), (True, False), (False, False)])
def test_without_initial_state_or_final_gradient(with_init, with_final):
    both_ways(5, (2, 150, 7), F32, BF16, True, with_init=with_init, with_final=with_final)
    both_ways(6, (150, 7), F32, F32, False, offsets=offsets_of([0, 70, 1, 79]), with_init=with_init, with_final=with_final)


PACKED = {
    "one": ([33], 0, 33),
    "empty ones everywhere": ([0, 0, 5, 0, 64, 0, 0, 59, 0], 0, 128),
    "only empty ones": ([0, 0, 0], 0, 0),
    "empty, with rows outside": ([0, 0], 3, 9),
    "rows outside on both sides": ([40, 0, 90, 3], 17, 200),
    "heads at the edges of waves and tiles": ([8, 8, 16, 32, 64, 128, 64, 1, 63, 128], 0, 512),
    "one long one between short ones": ([3, 1500, 2, 0, 11], 0, 1516),
    "single rows": ([1] * 300, 0, 300),
    "many, ragged": ([(i * 37) % 23 for i in range(200)], 5, 2300),
    "two long ones that meet inside a tile": ([700, 900], 0, 1600),
    "hundreds of empty ones in one place": ([3] + [0] * 200 + [1, 40] + [0] * 64 + [30] + [0] * 70, 0, 80),
}


@pytest.mark.parametrize("which", list(PACKED), ids=str)
@pytest.mark.parametrize("gate_t,x_t,wide", [(F32, F32, torch.int32), (F16, F16, torch.int64), (F32, BF16, torch.int32)], ids=name)
def test_packed(which, gate_t, x_t, wide):
    lengths, first, rows = PACKED[which]
    for channels in (3, 132):
        both_ways(len(which) + channels, (rows, channels), gate_t, x_t, log=channels == 3, offsets=offsets_of(lengths, first).to(wide))


def test_more_sequences_than_a_search_step():
    lengths = [i % 3 for i in range(5000)]  # two steps of the 64-way search
    both_ways(9, (sum(lengths), 2), F32, F32, False, offsets=offsets_of(lengths).int())


@pytest.mark.parametrize("channels", [4, 131, 132, 257])
def test_halves_of_a_projection_and_outputs_in_place(channels):
    shape = (2, 140, channels)
    gate, x, init, _, _ = inputs(11, shape, 2, BF16, BF16, False)
    ref = Recurrence(gate, x, init, None, False)
    for where in ("new", "x", "gate", "other"):
        both = put(torch.cat([gate, x], -1))
        g, v = both[..., :channels], both[..., channels:]
        keep = get(both)
        out = {"new": None, "x": v, "gate": g, "other": put(torch.full((2, 140, 2 * channels), 7.0, dtype=BF16))[..., channels:]}[where]
        got, final = thrust_amd.linear_scan(g, v, init=put(init), out=out)
        check(get(got), ref.out, ref.error_out, where)
        check(get(final), ref.final, ref.error_final, where)
        untouched = get(both)
        if where != "x":
            assert torch.equal(untouched[..., channels:], keep[..., channels:])
        if where != "gate":
            assert torch.equal(untouched[..., :channels], keep[..., :channels])
    # batches that are interleaved, rows apart
    v = put(x.transpose(0, 1).contiguous()).transpose(0, 1)
    got, _ = thrust_amd.linear_scan(put(gate), v, init=put(init))
    check(get(got), ref.out, ref.error_out, "interleaved")
    # one gate row for all batches
    got, _ = thrust_amd.linear_scan(put(gate[:1]).expand(shape), put(x), init=put(init))
    ref1 = Recurrence(gate[:1].expand(shape), x, init, None, False)
    check(get(got), ref1.out, ref1.error_out, "expanded")


@pytest.mark.parametrize("channels", [3, 133, 260])
def test_gradient_of_halves_and_of_interleaved_batches(channels):
    shape = (2, 150, channels)
    gate, x, init, grad_out, grad_final = inputs(21, shape, 2, F16, F16, False)
    ref = Recurrence(gate, x, init, None, False).gradient(grad_out, grad_final)
    both = put(torch.cat([gate, x], -1))
    g, v = both[..., :channels], both[..., channels:]
    d = put(grad_out.transpose(0, 1).contiguous()).transpose(0, 1)
    states = thrust_amd.linear_scan(g, v, init=put(init), return_states=True)[2]
    grads = thrust_amd.linear_scan_backward(d, g, v, states, init=put(init), grad_final=put(grad_final))
    assert all(t.is_contiguous() for t in grads)
    check(get(grads[0]), ref.grad_gate, ref.error_gate, "grad_gate")
    check(get(grads[1]), ref.grad_x, ref.error_x, "grad_x")
    check(get(grads[2]), ref.grad_init, ref.error_init, "grad_init")


@pytest.mark.parametrize("channels", [5, 131, 260])
def test_packed_in_place(channels):
    offsets = offsets_of([90, 0, 200, 7], 11)
    gate, x, init, _, _ = inputs(22, (330, channels), 4, F32, F32, True)
    ref = Recurrence(gate, x, init, offsets, True)
    for where in ("x", "gate"):
        both = put(torch.cat([gate, x], -1))
        g, v = both[..., :channels], both[..., channels:]
        out = v if where == "x" else g
        _, final = thrust_amd.linear_scan(g, v, init=put(init), offsets=put(offsets), log_gate=True, out=out)
        got, was = get(out), x if where == "x" else gate
        check(got[11:308], ref.out[0, 11:308], ref.error_out[0, 11:308], where)
        assert torch.equal(got[:11], was[:11]) and torch.equal(got[308:], was[308:])
        check(get(final), ref.final, ref.error_final, "final")


def test_unaligned_views():
    shape = (1, 70, 135)
    gate, x, init, grad_out, grad_final = inputs(12, shape, 1, BF16, BF16, False)
    ref = Recurrence(gate, x, init, None, False).gradient(grad_out, grad_final)

    def off(t):
        return put(torch.cat([torch.zeros(1, dtype=t.dtype), t.flatten()]))[1:].view(shape)
    out, _, states = thrust_amd.linear_scan(off(gate), off(x), init=put(init), return_states=True)
    check(get(out), ref.out, ref.error_out, "out")
    grads = thrust_amd.linear_scan_backward(off(grad_out), off(gate), off(x), states, init=put(init), grad_final=put(grad_final))
    check(get(grads[0]), ref.grad_gate, ref.error_gate, "grad_gate")
    check(get(grads[1]), ref.grad_x, ref.error_x, "grad_x")


def test_rows_outside_are_left_or_cleared():
    shape, offsets = (200, 133), offsets_of([50, 60], 30).int()
    gate, x, init, _, _ = inputs(13, shape, 2, F32, F16, False)
    out = put(torch.full(shape, 3.0, dtype=F16))
    forward(gate, x, init, offsets, False, out=out)
    got = get(out)
    assert (got[:30] == 3).all() and (got[140:] == 3).all()
    assert (get(forward(gate, x, init, offsets, False)[0])[140:] == 0).all()
    x[:30] = float("nan")  # what lies outside does not matter
    gate[140:] = float("inf")
    ref = Recurrence(gate, x, init, offsets, False)
    out, final = forward(gate, x, init, offsets, False)
    check(get(out)[30:140], ref.out[0, 30:140], ref.error_out[0, 30:140], "out")
    check(get(final), ref.final, ref.error_final, "final")


@pytest.mark.parametrize("x_t", [F32, BF16], ids=name)
def test_infinities_and_nans_stay_in_their_sequence_and_channel(x_t):
    lengths = [150, 200, 0, 300, 70]
    offsets = offsets_of(lengths).int()
    gate, x, init, grad_out, grad_final = inputs(14, (720, 130), 5, x_t, x_t, False)
    x[160, 3], gate[170, 5], init[1, 7], x[349, :9] = float("nan"), float("inf"), float("-inf"), float("inf")
    grad_out[200, 11], grad_final[1, 13] = float("nan"), float("inf")
    clean_x, clean_gate, clean_init, clean_out, clean_final = (t.clone() for t in (x, gate, init, grad_out, grad_final))
    clean_x[150:350], clean_gate[150:350], clean_init[1], clean_out[150:350], clean_final[1] = 1, 0.5, 0, 0, 0
    results = []
    for g, v, i, d, f in ((gate, x, init, grad_out, grad_final), (clean_gate, clean_x, clean_init, clean_out, clean_final)):
        out, final, states = forward(g, v, i, offsets, False, return_states=True)
        grads = thrust_amd.linear_scan_backward(put(d), put(g), put(v), states, init=put(i), grad_final=put(f), offsets=put(offsets))
        results.append([get(t) for t in (out, final, *grads)])
    rows = torch.ones(720, dtype=torch.bool)
    rows[150:350] = False
    sequences = torch.tensor([0, 2, 3, 4])
    for k, (a, b) in enumerate(zip(*results)):
        keep = sequences if k in (1, 4) else rows
        assert torch.isfinite(a[keep]).all() and torch.equal(a[keep], b[keep])
    ref = Recurrence(gate, x, init, offsets, False)
    out = results[0][0]
    # what follows is not finite either (NaN for an infinite state once the product of the gates behind it underflows)
    assert torch.equal(torch.isfinite(out), torch.isfinite(ref.out[0].to(x_t)))


def test_gates_of_zero_and_one_and_log_gates_of_minus_infinity():
    shape = (1, 300, 5)
    gate, x, init, grad_out, grad_final = inputs(15, shape, 1, F32, F32, False)
    gate[:, 100] = 0
    gate[:, 200:] = 1
    for log in (False, True):
        g = gate.abs().log() if log else gate.abs()
        ref = Recurrence(g, x, init, None, log).gradient(grad_out, grad_final)
        out, final, states = forward(g, x, init, None, log, return_states=True)
        check(get(out), ref.out, ref.error_out, "out")
        grads = thrust_amd.linear_scan_backward(put(grad_out), put(g), put(x), states, init=put(init), grad_final=put(grad_final), log_gate=log)
        check(get(grads[0]), ref.grad_gate, ref.error_gate, "grad_gate")
        check(get(grads[1]), ref.grad_x, ref.error_x, "grad_x")


def test_nothing_to_do():
    for shape, sequences in (((0, 5, 3), 0), ((2, 0, 3), 2), ((2, 5, 0), 2)):
        gate, x, init, grad_out, grad_final = inputs(16, shape, sequences, F32, F32, False)
        out, final, states = forward(gate, x, init, None, False, return_states=True)
        assert out.shape == shape
        if shape[1] == 0:
            assert torch.equal(get(final), init)
        grads = thrust_amd.linear_scan_backward(put(grad_out), put(gate), put(x), states, init=put(init), grad_final=put(grad_final))
        if shape[1] == 0:
            assert torch.equal(get(grads[2]), grad_final)
    gate, x, init, _, _ = inputs(16, (4, 3), 0, F32, F32, False)
    out, final = forward(gate, x, init, torch.zeros(1, dtype=torch.int32), False)
    assert final.shape == (0, 3) and (get(out) == 0).all()  # no sequences: every row is outside


def test_results_do_not_vary():
    gate, x, init, grad_out, grad_final = inputs(17, (1, 3000, 70), 1, F32, F32, False)
    d = [put(t) for t in (gate, x, init, grad_out, grad_final)]
    first = None
    for _ in range(4):
        out, final, states = thrust_amd.linear_scan(d[0], d[1], init=d[2], return_states=True)
        grads = thrust_amd.linear_scan_backward(d[3], d[0], d[1], states, init=d[2], grad_final=d[4])
        now = [get(t) for t in (out, final, states, *grads)]
        assert first is None or all(torch.equal(a, b) for a, b in zip(first, now))
        first = now


def test_gradient_against_differences():
    """A central difference of a 64-bit loss along a random direction.  With step e its error is e^2 / 6 of the third derivative and
    2^-53 / e of the loss; the gradient's own is bounded element by element."""
    gate, x, init, grad_out, grad_final = inputs(18, (2, 40, 3), 2, F32, F32, False)
    states = forward(gate, x, init, None, False, return_states=True)[2]
    grads = thrust_amd.linear_scan_backward(put(grad_out), put(gate), put(x), states, init=put(init), grad_final=put(grad_final))
    g = torch.Generator().manual_seed(1)
    along = [torch.randn(t.shape, generator=g, dtype=torch.float64) for t in (gate, x, init)]

    def loss(e):
        r = Recurrence(*(t.double() + e * v for t, v in zip((gate, x, init), along)), None, False)
        return float((r.out * grad_out.double()).sum() + (r.final * grad_final.double()).sum())
    e = 1e-5
    third = abs(loss(2e-2) - 2 * loss(1e-2) + 2 * loss(-1e-2) - loss(-2e-2)) / (2 * 1e-6)
    difference = (loss(e) - loss(-e)) / (2 * e)
    got = sum(float((get(a).double() * v).sum()) for a, v in zip(grads, along))
    ref = Recurrence(gate, x, init, None, False).gradient(grad_out, grad_final)
    own = sum(float((b * v.abs()).sum()) for b, v in zip((ref.error_gate, ref.error_x, ref.error_init), along)) \
        + 2.0 ** -24 * sum(float((r.abs() * v.abs()).sum()) for r, v in zip((ref.grad_gate, ref.grad_x, ref.grad_init), along))
    assert abs(got - difference) <= own + 2 * e * e / 6 * third + 2.0 ** -53 / e * 1e3


class Scan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gate, x, init):
        out, final, states = thrust_amd.linear_scan(gate, x, init=init, return_states=True)
        ctx.save_for_backward(gate, x, init, states)
        return out, final

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_out, grad_final):
        gate, x, init, states = ctx.saved_tensors
        return thrust_amd.linear_scan_backward(grad_out.contiguous(), gate, x, states, init=init, grad_final=grad_final.contiguous())


def test_as_a_function_of_torch():
    """A model's layer: the two halves of a projection go in, a loss that sums comes back expanded."""
    gate, x, init, _, _ = inputs(19, (2, 90, 6), 2, F32, F32, True)
    leaf, h0 = put(torch.cat([gate, x], -1)).requires_grad_(), put(init).requires_grad_()
    with pytest.raises(ValueError):
        thrust_amd.linear_scan(*leaf.chunk(2, -1), init=h0)
    g, v = leaf.chunk(2, -1)
    out, final = Scan.apply(g.exp(), v, h0)
    (out.sum() + 3 * final.sum()).backward()
    ref = Recurrence(gate, x, init, None, True).gradient(torch.ones_like(x), torch.full_like(init, 3))
    # torch's exp and its gradient add at most two units in the last place to a gate's factor and one product: covered twice over by the
    # bound for logarithms, whose own exp is counted in it
    check(get(leaf.grad)[..., :6], ref.grad_gate, 2 * ref.error_gate, "gate")
    check(get(leaf.grad)[..., 6:], ref.grad_x, 2 * ref.error_x, "x")
    check(get(h0.grad), ref.grad_init, 2 * ref.error_init, "init")


# ---------------------------------------------------------------------------------------
# The step
# ---------------------------------------------------------------------------------------
def step_reference(gate, x, state, slots, log):
    a = gate.double().exp() if log else gate.double()
    state, out = state.double().clone(), torch.zeros(x.shape, dtype=torch.float64)
    error_state, error = torch.zeros_like(state), torch.zeros_like(out)
    for i, s in enumerate(slots):
        if 0 <= s < state.shape[0]:
            size = (a[i] * state[s]).abs() + x[i].double().abs()
            error_state[s] = a[i].abs() * error_state[s] + 2.0 ** -24 * (6 if log else 4) * size
            state[s] = a[i] * state[s] + x[i].double()
            out[i], error[i] = state[s], error_state[s]
    return out, state, error, error_state


@pytest.mark.parametrize("gate_t,x_t", TYPES, ids=name)
@pytest.mark.parametrize("batch,channels", [(1, 1), (3, 5), (7, 132), (2, 1030), (130, 4)])
def test_step(gate_t, x_t, batch, channels):
    log = channels % 2 == 0
    gate, x, _, _, _ = inputs(20 + batch, (batch, channels), batch, gate_t, x_t, log)
    g = torch.Generator().manual_seed(3)
    state = torch.randn((batch + 9, channels), generator=g)
    for slots in (None, torch.randperm(batch + 9, generator=g)[:batch].int()):
        on = put(state)
        out = thrust_amd.linear_scan_step(put(gate), put(x), on, slots=put(slots), log_gate=log)
        want, after, error, error_state = step_reference(gate, x, state, range(batch) if slots is None else slots.tolist(), log)
        check(get(out), want, error, "out")
        check(get(on), after, error_state, "state")


def test_step_padding_and_rows_of_one_slot():
    gate, x, _, _, _ = inputs(30, (140, 9), 140, F32, F32, False)
    g = torch.Generator().manual_seed(4)
    state = torch.randn((20, 9), generator=g)
    slots = torch.randint(-2, 22, (140,), generator=g).int()  # every slot several times, and ids outside
    slots[5], slots[6] = 2 ** 31 - 1, -2 ** 31
    on = put(state)
    out = get(thrust_amd.linear_scan_step(put(gate), put(x), on, slots=put(slots)))
    want, after, error, error_state = step_reference(gate, x, state, slots.tolist(), False)
    check(out, want, error, "out")
    check(get(on), after, error_state, "state")
    assert (out[(slots < 0) | (slots >= 20)] == 0).all()


def test_step_of_a_large_batch_with_rows_of_one_slot():
    gate, x, _, _, _ = inputs(32, (2500, 5), 2500, F32, F32, False)
    g = torch.Generator().manual_seed(6)
    state = torch.randn((3000, 5), generator=g)
    slots = torch.randperm(3000, generator=g)[:2500].int()
    slots[2400], slots[7], slots[1300], slots[1301], slots[2499] = slots[3], slots[1027], slots[1299], slots[1299], -1
    on = put(state)
    out = thrust_amd.linear_scan_step(put(gate), put(x), on, slots=put(slots))
    want, after, error, error_state = step_reference(gate, x, state, slots.tolist(), False)
    check(get(out), want, error, "out")
    check(get(on), after, error_state, "state")


def test_step_is_a_scan_of_one_row_and_takes_halves_of_a_projection():
    gate, x, init, _, _ = inputs(31, (6, 132), 6, BF16, BF16, False)
    both = put(torch.cat([gate, x], -1))
    g, v = both[:, :132], both[:, 132:]
    state = put(init)
    out = thrust_amd.linear_scan_step(g, v, state)
    want, final = thrust_amd.linear_scan(g.unsqueeze(1), v.unsqueeze(1), init=put(init))
    assert torch.equal(get(out), get(want)[:, 0]) and torch.equal(get(state), get(final))
    state = put(init)
    assert thrust_amd.linear_scan_step(g, v, state, out=v) is v
    assert torch.equal(get(v), get(want)[:, 0])


# ---------------------------------------------------------------------------------------
# On the device
# ---------------------------------------------------------------------------------------
@pytest.mark.needs_device
def test_training_in_a_graph():
    gate, x, init, grad_out, grad_final = inputs(40, (2, 700, 261), 2, F32, BF16, True)
    d = [put(t) for t in (gate, x, init, grad_out, grad_final)]

    def one():
        out, final, states = thrust_amd.linear_scan(d[0], d[1], init=d[2], log_gate=True, return_states=True)
        return (out, final) + thrust_amd.linear_scan_backward(d[3], d[0], d[1], states, init=d[2], grad_final=d[4], log_gate=True)
    one()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):  # two graphs, each with storage of its own
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs = one()
        graphs.append((g, outs))
    for r in range(4):
        fresh = inputs(50 + r, (2, 700, 261), 2, F32, BF16, True)
        for a, b in zip(d, fresh):
            a.copy_(b)
        want = [t.clone() for t in one()]
        torch.cuda.synchronize()
        for g, outs in graphs:
            g.replay()
            one()  # eager work behind it
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(outs, want))


@pytest.mark.needs_device
def test_step_in_a_graph():
    gate, x, _, _, _ = inputs(42, (40, 1030), 40, F32, BF16, True)
    state = torch.randn((64, 1030), generator=torch.Generator().manual_seed(8))
    d = [put(t) for t in (gate, x, state)]
    slots = put(torch.arange(40).int())
    thrust_amd.linear_scan_step(d[0], d[1], d[2], slots=slots, log_gate=True)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = thrust_amd.linear_scan_step(d[0], d[1], d[2], slots=slots, log_gate=True)
    g = torch.Generator().manual_seed(9)
    for r in range(4):
        new = torch.randint(-3, 64, (40,), generator=g).int()  # padded rows, and rows of one slot
        slots.copy_(new)
        d[2].copy_(state)
        graph.replay()
        torch.cuda.synchronize()
        want, after, error, error_state = step_reference(gate, x, state, new.tolist(), True)
        check(get(out), want, error, "out")
        check(get(d[2]), after, error_state, "state")


@pytest.mark.needs_device
def test_streams():
    gate, x, init, _, _ = inputs(41, (1, 5000, 300), 1, F32, F32, False)
    d = [put(t) for t in (gate, x, init)]
    want = thrust_amd.linear_scan(d[0], d[1], init=d[2])[0]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    for k in range(9):
        with torch.cuda.stream(streams[k % 3]):
            outs.append(thrust_amd.linear_scan(d[0], d[1], init=d[2])[0])
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


@pytest.mark.needs_device
def test_more_than_2_to_the_32_elements():
    rows, channels = (1 << 20) + 700, 4100
    x = torch.ones((1, rows, channels), dtype=BF16, device="cuda")
    gate = torch.full((1, rows, channels), 0.5, dtype=BF16, device="cuda")
    init = torch.full((1, channels), 1e30, device="cuda")
    out, final, states = thrust_amd.linear_scan(gate, x, init=init, return_states=True)
    assert (out[0, 1000::1777] == 2).all() and (out[0, -300:] == 2).all() and (final == 2).all()
    assert states.shape == (1, -(-rows // 64), channels) and (states[0, 40:] == 2).all()
    grad_out = torch.zeros_like(x)
    grad_out[0, -1] = 1
    del out
    grad_gate, grad_x, grad_init = thrust_amd.linear_scan_backward(grad_out, gate, x, states, init=init)
    want = torch.tensor([2.0 ** -k for k in range(100)], device="cuda")  # powers of two: exact
    assert torch.equal(grad_x[0, -100:].flip(0).float(), want[:, None].expand(-1, channels))
    assert torch.equal(grad_gate[0, -100:].flip(0).float(), 2 * want[:, None].expand(-1, channels))
    assert (grad_init == 0).all() and (grad_x[0, : rows // 2: 1009] == 0).all()


@pytest.mark.needs_device
def test_no_wait_was_given_up():
    count = ctypes.c_ulonglong(7)
    capi.check(capi.lib().thrust_cdna4_lookback_timeouts(ctypes.byref(count)), "lookback_timeouts")
    assert count.value == 0
    gpu_util.synchronize()


# ---------------------------------------------------------------------------------------
# Gates whose products leave the range of 32 bits where the states do not
# ---------------------------------------------------------------------------------------
# name: rows, {row: gate} (1 elsewhere), initial state, gradient of the final one.  Every state of the rows one after the other, and
# every gradient, is a normal number of 32 bits; the product of some of the gates is not.
RANGES = {
    "over, along tiles": (900, {t: 2.0 for t in range(512, 640)}, 1e-20, 1e-20),
    "under, along tiles": (900, {t: 0.5 for t in range(512, 672)}, 1e30, 1e30),
    "over, along wavefronts": (70, {t: 64.0 for t in range(8, 38)}, 1e-25, 1e-25),
    "under, along wavefronts": (70, {t: 2.0 ** -6 for t in range(8, 38)}, 1e25, 1e25),
    "over, along rows": (5, {1: 1e20, 2: 1e20}, 1e-30, 1e-18),
    "under, along rows": (5, {1: 1e-25, 2: 1e-20}, 1e30, 1e18),
    "over and back": (1500, {**{t: 8.0 for t in range(100, 160)}, **{t: 0.125 for t in range(1300, 1350)}}, 1e-25, 1e20),
    "under and back": (1500, {**{t: 0.125 for t in range(100, 160)}, **{t: 8.0 for t in range(1300, 1350)}}, 1e25, 1e-10),
    "over and back in a wavefront": (16, {2: 1e18, 3: -1e18, 4: 1e18, 5: 1e-17, 6: 1e-18, 7: 1e-18}, 1e-27, 1e20),
    "the smallest gate": (200, {150: 2.0 ** -133, 151: 0.5}, 1e30, 1e5),
    "past a super-group": (9100, {t: 0.5 for t in range(8100, 8280)}, -1e35, 1e25),
}


@pytest.mark.parametrize("which", list(RANGES), ids=str)
@pytest.mark.parametrize("gate_t,x_t,channels,log", [(F32, F32, 4, False), (BF16, BF16, 132, False), (F32, BF16, 132, True), (F32, F32, 130, False)], ids=name)
def test_products_of_gates_out_of_range(which, gate_t, x_t, channels, log):
    rows, gates, first, last = RANGES[which]
    if channels > 4 and rows > 1600:
        channels = 129
    gate = torch.ones(1, rows, channels, dtype=torch.float64)
    for t, a in gates.items():
        gate[0, t] = a
    if log:
        gate = gate.abs().log()
    gate = gate.to(gate_t)
    x, grad_out = torch.zeros(1, rows, channels, dtype=x_t), torch.zeros(1, rows, channels, dtype=x_t)
    scale = 1 + torch.arange(channels) / 512.0
    init, grad_final = (first * scale)[None].float(), (last * scale)[None].float()
    ref = Recurrence(gate, x, init, None, log).gradient(grad_out, grad_final)
    for v in (ref.out, ref.grad_x, ref.grad_x * ref.a, ref.grad_x * ref.before, ref.grad_gate):  # what is said above
        assert v.abs().min() >= 2.0 ** -126 and v.abs().max() < 2.0 ** 128
    d = [put(t) for t in (gate, x, init, grad_out, grad_final)]
    out, final, states = thrust_amd.linear_scan(d[0], d[1], init=d[2], log_gate=log, return_states=True)
    check(get(out), ref.out, ref.error_out, "out")
    check(get(final), ref.final, ref.error_final, "final")
    grads = thrust_amd.linear_scan_backward(d[3], d[0], d[1], states, init=d[2], grad_final=d[4], log_gate=log)
    check(get(grads[1]), ref.grad_x, ref.error_x, "grad_x")
    check(get(grads[0]), ref.grad_gate, ref.error_gate, "grad_gate")
    check(get(grads[2]), ref.grad_init, ref.error_init, "grad_init")
    # the same as one of several packed sequences
    offsets = offsets_of([70, rows, 0, 33]).int()
    wide = (rows + 103, channels)
    g, v = torch.full(wide, float(0 if log else 1)).to(gate_t), torch.ones(wide).to(x_t)
    g[70:70 + rows], v[70:70 + rows] = gate[0], 0
    starts = torch.ones(4, channels)
    starts[1] = init[0]
    out, final = forward(g, v, starts, offsets, log)
    check(get(out)[70:70 + rows], ref.out[0], ref.error_out[0], "packed")
    check(get(final)[1], ref.final[0], ref.error_final[0], "packed, final")


def test_infinite_and_zero_states_meet_products_out_of_range():
    """An infinite state stays infinite under gates that are not zero, and a zero one zero under finite ones."""
    for a in (2.0 ** -6, 64.0):
        gate, x = torch.full((1, 700, 4), a), torch.zeros(1, 700, 4)
        out, final = forward(gate, x, torch.tensor([[float("inf"), 0.0, -float("inf"), float("nan")]]), None, False)
        got = torch.cat([get(out)[0], get(final)])
        assert (got[:, 0] == float("inf")).all() and (got[:, 1] == 0).all() and (got[:, 2] == -float("inf")).all() and got[:, 3].isnan().all()


def test_torch_is_told_what_is_written():
    """A tensor saved for somebody's backward pass and then written by a call is found out, as after any operation of torch in place."""
    gate, x, init, _, _ = inputs(60, (2, 30, 5), 2, F32, F32, False)
    g, v, state = put(gate), put(x), put(init)
    weight = put(torch.ones(5)).requires_grad_()
    loss = (v * weight).sum()
    was = g._version, v._version
    thrust_amd.linear_scan(g, v, out=v)
    assert g._version == was[0] and v._version > was[1]
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    loss = (state * weight).sum()
    rows, out = put(gate[:, 0]), put(x[:, 0])
    was = rows._version, state._version, out._version
    thrust_amd.linear_scan_step(rows, out, state, out=out)
    assert rows._version == was[0] and state._version > was[1] and out._version > was[2]
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


# batches that are large enough for four vectors a thread: two workgroups to each of 256 compute units, or of the emulator's 8
WIDE = [(20, c) if EMULATED else (b, c) for b, c in ((600, 1030), (600, 2051), (520, 4096), (300, 4101), (270, 8190))]


@pytest.mark.parametrize("gate_t,x_t", [(F32, F32), (F16, F16), (F32, BF16)], ids=name)
@pytest.mark.parametrize("batch,channels", WIDE, ids=str)
def test_step_of_a_large_batch_of_wide_rows(batch, channels, gate_t, x_t):
    """Every vector of a thread, the partial one behind the last whole one, several blocks of channels; rows of one slot and padded ones."""
    log = channels % 2 == 0
    gate, x, _, _, _ = inputs(70 + batch, (batch, channels), batch, gate_t, x_t, log)
    g = torch.Generator().manual_seed(channels)
    state = torch.randn((batch + 5, channels), generator=g)
    slots = torch.randperm(batch + 5, generator=g)[:batch].int()
    slots[3], slots[7], slots[11], slots[batch - 1] = -1, slots[1], slots[1], slots[0]
    want, after, error, error_state = step_reference(gate, x, state, slots.tolist(), log)
    wide = put(torch.full((batch, 2 * channels + 3), 7.0).to(x_t))
    for rows in ("apart", "halves of a projection"):
        on, a, b = put(state), put(gate), put(x)
        if rows != "apart" and gate_t == x_t:
            both = put(torch.cat([gate, x], -1))
            a, b = both[:, :channels], both[:, channels:]
        out = None if rows == "apart" else wide[:, channels + 1:-2]
        got = thrust_amd.linear_scan_step(a, b, on, slots=put(slots), log_gate=log, out=out)
        check(get(got), want, error, "out")
        check(get(on), after, error_state, "state")
    assert (get(wide)[:, : channels + 1] == 7).all() and (get(wide)[:, -2:] == 7).all()
    on = put(state)
    assert thrust_amd.linear_scan_step(a, b, on, slots=put(slots), log_gate=log, out=b) is b  # in place
    check(get(b), want, error, "in place")
    check(get(on), after, error_state, "state")


def test_a_state_between_the_rows_of_an_input():
    """Ranges that meet without an element in common are no overlap."""
    gate, x, _, _, _ = inputs(80, (3, 4), 3, F32, F32, False)
    init = torch.randn((2, 4), generator=torch.Generator().manual_seed(1))
    buffer = torch.zeros(3, 12)
    buffer[:, :4] = x
    buffer[1, 4:] = init.flatten()
    on = put(buffer)
    state = on.flatten()[16:24].view(2, 4)
    slots = torch.tensor([1, 0, 1], dtype=torch.int32)
    out = thrust_amd.linear_scan_step(put(gate), on[:, :4], state, slots=put(slots))
    want, after, error, error_state = step_reference(gate, x, init, slots.tolist(), False)
    check(get(out), want, error, "out")
    check(get(state), after, error_state, "state")
    assert torch.equal(get(on)[:, :4], x)
