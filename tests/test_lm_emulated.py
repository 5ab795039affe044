"""The tests of the linear recurrence and the page cache run WITHOUT a GPU, on the lockstep emulator
(tests/test_emulated_kernels.py says what that shows): one workgroup at a time with every buffer ending
at an inaccessible page, and several workgroups in flight in seeded interleavings."""
import pytest

from test_emulated_kernels import emulated_library, run_session  # noqa: F401


def test_nothing_outside_the_ranges(emulated_library):  # noqa: F811
    print(run_session(["tests/test_linear_scan_gpu.py", "tests/test_pages_gpu.py"], guard=True))


@pytest.mark.parametrize("resident", ["7:3", "16:21"])
def test_tiles_in_flight(emulated_library, resident):  # noqa: F811
    print(run_session(["tests/test_linear_scan_gpu.py", "tests/test_pages_gpu.py"], resident=resident,
                      extra=["-k", "many_tiles or past_super or packed or vary or fork or resize or compact or life"]))


@pytest.mark.parametrize("resident", ["1", "40:9"])
def test_waits_that_are_given_up(emulated_library, resident):  # noqa: F811
    print(run_session(["tests/test_zw_recurrence_timeout_gpu.py"], resident=resident))
