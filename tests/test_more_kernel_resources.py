"""Registers and LDS of the kernels for shared and selected pages, bounds and
drafted tokens: launches count on the workgroups that a compute unit holds."""
import re

from epure.kernels import _abi
from test_kernel_resources import kernels
from test_paged_kernel_resources import workgroups

BF16, F16, E4M3, I8 = _abi.BF16, _abi.F16, _abi.E4M3, _abi.I8
TYPES = {("Bf16", BF16), ("F16", F16), *((q, c) for q in ("Bf16", "F16") for c in (E4M3, I8))}


def found(pattern):
    out = {}
    for name, k in kernels(_abi.LIB_PATH).items():
        m = re.search(pattern, name)
        if m:
            out[m.groups()] = k
    return out


def test_parts_fit_as_many_workgroups_as_the_plan_counts_on():
    """As the kernels that answer at once: one and two row tiles, five widths."""
    made = found(r"attend_parts_kernel<ep::Op(Bf16|F16), (\d+), (\d+), (\d+), (\d+)>")
    assert {(q, int(c)) for q, c, *_ in made} == TYPES and len(made) == 6 * 5 * 2
    for (_, code, _, columns, tiles), k in made.items():
        n = workgroups(int(columns), int(tiles), int(code) != I8)
        assert k[".vgpr_count"] <= 512 // n, k[".name"]
        assert k[".vgpr_spill_count"] == 0 and k[".private_segment_fixed_size"] == 0, k[".name"]
        assert k[".group_segment_fixed_size"] <= 160 * 1024 // n, k[".name"]


def test_lists_of_pages_fit_the_registers():
    """A list is cut for two workgroups a compute unit; heads past 192 values hold one."""
    made = found(r"attend_blocks_kernel<ep::Op(Bf16|F16), (\d+), (\d+), (\d+)>")
    assert {(q, int(c)) for q, c, *_ in made} == TYPES and len(made) == 6 * 5
    for (_, _, _, columns), k in made.items():
        n = 2 if int(columns) <= 12 else 1
        assert k[".vgpr_count"] <= 512 // n, k[".name"]
        assert k[".vgpr_spill_count"] == 0 and k[".private_segment_fixed_size"] == 0, k[".name"]
        assert k[".group_segment_fixed_size"] <= 160 * 1024 // n, k[".name"]


def test_shared_pages_through_lds_fit_two_workgroups():
    """kFrontOccupancy of attend_front.h, for the shared pages alone and with the others'.  Heads of 128 values take
    all registers and put up to three more away."""
    made = found(r"front(_tails)?_kernel<ep::Op(Bf16|F16), (\d+), (\d+)>")
    assert {(q, int(c)) for _, q, c, _ in made} == TYPES and len(made) == 2 * 6 * 3
    for (_, _, _, steps), k in made.items():
        away = 3 if int(steps) == 4 else 0
        assert k[".vgpr_count"] <= 512 // 2, k[".name"]
        assert k[".vgpr_spill_count"] <= away and k[".private_segment_fixed_size"] <= 4 * away, k[".name"]
        assert k[".group_segment_fixed_size"] <= 160 * 1024 // 2, k[".name"]


def test_small_kernels_keep_everything_in_registers():
    made = found(r"((?:bounds|score|choose|select|sum|pick|join_parts|join_blocks)_kernel.*)")
    assert len(made) == 12 + 2 + 1 + 2 + 6 + 3 + 2 + 2
    for k in made.values():
        assert k[".vgpr_spill_count"] == 0 and k[".private_segment_fixed_size"] == 0, k[".name"]
        assert k[".vgpr_count"] <= 128, k[".name"]
        assert k[".group_segment_fixed_size"] <= 64 * 1024, k[".name"]
