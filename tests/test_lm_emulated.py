"""The tests of the linear recurrence and the page cache run WITHOUT a GPU, on the lockstep emulator
(tests/test_emulated_kernels.py says what that shows): one workgroup at a time with every buffer ending
at an inaccessible page, and several workgroups in flight in seeded interleavings."""
import os
import subprocess

import pytest

from test_emulated_kernels import EMU_DIR, emulated_library, run_session  # noqa: F401


def test_nothing_outside_the_ranges(emulated_library):  # noqa: F811
    print(run_session(["tests/test_linear_scan_gpu.py", "tests/test_pages_gpu.py"], guard=True))


@pytest.mark.parametrize("resident", ["7:3", "16:21"])
def test_tiles_in_flight(emulated_library, resident):  # noqa: F811
    print(run_session(["tests/test_linear_scan_gpu.py", "tests/test_pages_gpu.py"], resident=resident,
                      extra=["-k", "many_tiles or past_super or packed or vary or fork or resize or compact or life"]))


@pytest.mark.parametrize("resident", ["1", "40:9"])
def test_waits_that_are_given_up(emulated_library, resident):  # noqa: F811
    print(run_session(["tests/test_zw_recurrence_timeout_gpu.py"], resident=resident))


@pytest.mark.parametrize("resident", ["1", "6:4"])
def test_no_data_race_between_wavefronts(resident):
    """Under ThreadSanitizer, which sees every wavefront as a thread and workgroup barriers, the ends of launches and atomics as the
    only ordering (test_emulated_kernels.py shows that it reports what it should)."""
    r = subprocess.run(["make", "-C", EMU_DIR, "-j8", "build/tsan/race_lm"], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout[-3000:] + r.stderr[-3000:]
    env = dict(os.environ, TSAN_OPTIONS="halt_on_error=1", THRUST_CDNA4_EMULATED_RESIDENT=resident)
    p = subprocess.run([os.path.join(EMU_DIR, "build", "tsan", "race_lm")], env=env, capture_output=True, text=True, timeout=900)
    out = p.stdout + p.stderr
    assert p.returncode == 0 and "race_lm: done" in out and "ThreadSanitizer" not in out, out[-4000:]


def test_the_measured_cases_at_small_sizes(emulated_library):  # noqa: F811
    print(run_session(["tests/test_lm_cases_gpu.py"], resident="5:8"))
