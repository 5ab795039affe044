"""The cases of perf/operators.py at small sizes: its plain forms, its exact values and the calls of the package say the same."""
import importlib.util
import os
import random

import pytest
import torch

from conftest import EMULATED, ROOT
from lm_util import Recurrence, check

spec = importlib.util.spec_from_file_location("perf_operators", os.path.join(ROOT, "perf", "operators.py"))
operators = importlib.util.module_from_spec(spec)
spec.loader.exec_module(operators)

MOST = dict(batch=3, rows=150, channels=70, packed=7, slots=12, pools=3, pages=60, page=13, sequences=16, max_pages=6, pairs=5)


def small(case):
    case = {k: min(v, MOST[k]) if k in MOST else v for k, v in case.items()}
    return dict(case, batch=1) if case.get("packed") else case


_rng = random.Random(5)
CASES = [small(c) for c in operators.listed()] + [dict(small(operators.draw(_rng)), name=f"drawn {k}") for k in range(25)]


def both(monkeypatch, case, own, device):
    monkeypatch.setattr(operators, "own", own)
    monkeypatch.setattr(operators, "DEVICE", device)
    seed = sum(map(ord, case["name"]))
    state = operators.prepare(case, seed)
    ref = None
    if case["op"] in ("scan", "grad"):
        args = [None if state[k] is None else state[k].cpu() for k in ("gate", "x", "init", "offsets")]
        ref = Recurrence(*args, case["log"])
        if case["op"] == "grad":
            ref.gradient(state["grad_out"].cpu(), state["grad_final"].cpu())
    want = operators.exact(case, seed)
    got = operators.run(state)
    assert got.keys() == want.keys()
    for k in want:
        if k == "pools":
            assert all(torch.equal(a.double().cpu(), b.cpu()) for a, b in zip(got[k], want[k]))
        elif not got[k].dtype.is_floating_point:
            assert got[k].dtype == want[k].dtype and torch.equal(got[k].cpu(), want[k].cpu()), k
        elif ref is None:  # a step: a product, a sum, exp, each within two half steps of 2^-24
            at = state["slots"].cpu().long()
            size = torch.zeros(case["slots"], case["channels"], dtype=torch.float64)
            a, x = state["gate"].cpu().double(), state["x"].cpu().double()
            before = operators.prepare(case, seed)["pool"].cpu().double()[at]
            size[at] = ((a.exp() if case["log"] else a) * before).abs() + x.abs()
            error = 6 * 2.0 ** -24 * size
            check(got[k].cpu(), want[k].cpu(), error if k == "pool" else error[at], k)
        else:
            mine = {"out": (ref.out, ref.error_out), "final": (ref.final, ref.error_final)}
            if case["op"] == "grad":
                mine.update(grad_gate=(ref.grad_gate, ref.error_gate), grad_x=(ref.grad_x, ref.error_x), grad_init=(ref.grad_init, ref.error_init))
            assert torch.allclose(want[k].cpu().reshape(mine[k][0].shape), mine[k][0], rtol=1e-10, atol=1e-13), k  # 150 rows in 64 bits
            check(got[k].cpu(), *mine[k], k)


@pytest.mark.skipif(EMULATED, reason="runs without a device")
@pytest.mark.parametrize("case", CASES, ids=lambda c: c["name"])
def test_plain_form(monkeypatch, case):
    both(monkeypatch, case, False, "cpu")


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=lambda c: c["name"])
def test_own(monkeypatch, case):
    both(monkeypatch, case, True, "cpu" if EMULATED else "cuda")
