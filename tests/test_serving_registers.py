"""What rotary positions, appending and attention over a paged cache count on, as the built library states it: nothing spilled, and two wavefronts of
attention on a SIMD but where keys, values, queries and sums fill the registers of one."""

import collections
import re

from tests.test_operator_registers import LDS, REGISTERS, _kernels


def test_wavefronts_on_a_simd_and_nothing_spilled():
    seen = collections.Counter()
    for k in _kernels():
        m = re.search(r"(attend_kernel|attend_join_kernel|append_kernel|rotary_kernel)I", k[".name"])
        if not m:
            continue
        seen[m[1]] += 1
        assert k[".vgpr_spill_count"] == 0 and k[".private_segment_fixed_size"] == 0, k[".name"]
        waves = 4
        if m[1] == "attend_kernel":
            nk, nv = map(int, re.search(r"ELi(\d)ELi(\d)ELb", k[".name"]).groups())
            waves = 1 if nv == 2 and nk > 4 else 2
        assert k[".vgpr_count"] * waves <= REGISTERS and k[".group_segment_fixed_size"] * waves <= LDS, k[".name"]
    assert seen == {"rotary_kernel": 18, "append_kernel": 8, "attend_join_kernel": 8, "attend_kernel": 128}
