"""Host checks of the row operators at the ends of what they take: calls that are refused before any device call."""

from __future__ import annotations

import pytest

from povs import _native

A = 64  # an address on every element's boundary
CALLS = {
    # name: (arguments, {place: size of the elements there})
    "povs_sample_v1": ([A, 0, 2, 8, 8, A, 8, A, 1.0, A, 0, A, 1.0, A, 0.0, A, 0, None],
                       {0: 4, 5: 8, 7: 4, 9: 4, 11: 4, 13: 4, 15: 8}),
    "povs_route_v1": ([A, 1, 2, 16, 16, A, 2, 0, 1, 1, 0, 0, 1.0, A, A, 0, None], {0: 2, 5: 4, 13: 4, 14: 4}),
    "povs_route_backward_v1": ([A, 2, 2, 16, 16, 2, 0, 0, 1.0, A, A, A, 0, None], {0: 2, 9: 4, 10: 4, 11: 2}),
    "povs_plan_rows_v1": ([A, 8, 1 << 20, 256, A, A, A, A, 1 << 30, 0, None], {0: 8, 4: 4, 5: 4, 6: 4, 7: 4}),
    "povs_dispatch_rows_v1": ([A, 4, 16, 16, A, 2, A, A, 8, 0, None], {4: 4, 6: 4}),
    "povs_combine_rows_v1": ([A, 0, 8, 16, 16, A, 4, 2, A, A, 0, None], {0: 4, 5: 4, 8: 4, 9: 4}),
    "povs_combine_backward_v1": ([A, A, 1, 8, 16, 16, A, 4, 2, A, A, A, A, 0, None],
                                 {0: 2, 1: 2, 6: 4, 9: 4, 10: 4, 11: 2, 12: 4}),
}


@pytest.mark.parametrize("name,place,size", [(n, p, s) for n, (_, places) in CALLS.items() for p, s in places.items()])
def test_pointers_off_their_elements_are_refused(name, place, size):
    lib = _native.load()
    for off in range(1, size):
        args = list(CALLS[name][0])
        args[place] = A + off
        assert getattr(lib, name)(*args) == -1
        assert b"not aligned" in lib.povs_last_error_string()
