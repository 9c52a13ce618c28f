"""The sizes of test_gpu_linear_kinds.py reach every kernel of linear, cut and whole, on a GPU of 256 CUs: by the rule's own tables, so that new ones cannot leave a kernel untested."""
import pytest

import test_gpu_linear_kinds as gpu
from linear_rule import a_float_a_load, choose, kinds, launches


@pytest.mark.parametrize("bits", [16, 32])
def test_every_kernel_is_reached(bits):
    table = kinds(bits)
    assert len(table) == (5 if bits == 16 else 3)
    parts = (1, 2) if bits == 16 else (1,)
    want = {("forward", k, cut) for k in range(len(table)) for cut in (False, True)}
    want |= {("both", p, k) for p in parts for k in range(len(table))}
    want |= {(role, p, k, cut) for role in ("grad_x", "grad_w", "both, grad_x", "both, grad_w") for p in parts for k in range(len(table)) for cut in (False, True)}
    for rounded in (False, True):
        have = set()
        for size in gpu.SIZES[bits]:
            for p in parts:
                have |= launches(*gpu.rounded(size) if rounded else size, bits, p)
        # (two products of kind 2 with grad_x's cut are one size in 40 000; the same kernel runs with grad_w's cut, and its sums' launch for grad_x with other kinds)
        assert want - have <= {("both, grad_x", 1, 2, True)}, sorted(want - have)


def test_floats_that_begin_anywhere():
    """Read one by one and laid out anew, by every kind of tiles."""
    have = {(choose(*size, 32)[0], a_float_a_load(*size)) for size in gpu.SIZES[32]}
    assert have >= {(k, one) for k in range(3) for one in (False, True)}, sorted(have)
