"""Registers and LDS of the built attention kernels: the plan of a call counts
on as many workgroups a compute unit as attend_occupancy says."""
import re

from epure.kernels import _abi
from test_kernel_resources import kernels

BF16, F16, E4M3, I8 = _abi.BF16, _abi.F16, _abi.E4M3, _abi.I8


def workgroups(columns, tiles, lookout):
    """Of four waves, resident on a compute unit (csrc/attend_kernel.h, attend_occupancy)."""
    if columns == 4:
        return 3 if tiles == 1 else 2
    return 2 if columns == 8 or (columns == 12 and tiles == 1 and not lookout) else 1


def test_attention_kernels_fit_as_many_workgroups_as_the_plan_counts_on():
    """Four SIMDs of 512 registers a lane (accumulators counted among them), a wave of each workgroup on every
    one; 160 KiB of LDS; nothing through memory."""
    found = {}
    for name, k in kernels(_abi.LIB_PATH).items():
        m = re.search(r"attend_kernel<ep::Op(Bf16|F16), (\d+), (\d+), (\d+), (\d+), (true|false)>", name)
        if m:
            found[m.groups()] = k
    types = {(q, c) for q, c, *_ in found}
    assert types == {("Bf16", str(BF16)), ("F16", str(F16)), *((q, str(c)) for q in ("Bf16", "F16") for c in (E4M3, I8))}
    # 64, 96 (16-bit rows), 128, 144 and 192, up to 192, up to 256 values; one token, several, two row tiles
    assert len(found) == 3 * (2 * 6 + 4 * 5)
    for (_, code, _, columns, tiles, ragged), k in found.items():
        n = workgroups(int(columns), int(tiles), ragged == "true" and int(code) != I8)
        assert k[".vgpr_count"] <= 512 // n, k[".name"]
        assert k[".vgpr_spill_count"] == 0 and k[".private_segment_fixed_size"] == 0, k[".name"]
        assert k[".group_segment_fixed_size"] <= 160 * 1024 // n, k[".name"]
