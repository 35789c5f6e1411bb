"""What the products' plan counts on, as the built library states it: workgroups of each tile on a compute unit, and nothing spilled."""

import re
import struct

import msgpack

from miles_amd import _lib

LDS, REGISTERS = 160 * 1024, 512        # of a compute unit, and of a lane on a SIMD with one wavefront


def _kernels():
    data = open(_lib.lib_path(), "rb").read()
    at = data.find(b"AMDGPU\0")
    while at >= 0:
        name_size, size, kind = struct.unpack_from("<III", data, at - 12)
        if (name_size, kind) == (7, 32):        # NT_AMDGPU_METADATA
            yield from msgpack.unpackb(data[at + 8:at + 8 + size], strict_map_key=False)["amdhsa.kernels"]
        at = data.find(b"AMDGPU\0", at + 1)


def test_workgroups_of_a_tile_on_a_compute_unit():
    """Four wavefronts each, one on every SIMD: 256 x 256 alone, 128 x 128 two, 128 x 64 two and in the weight gradient three."""
    seen = 0
    for k in _kernels():
        m = re.search(r"gemm_kernelILi\dELi\dELi(\d)ELi(\d+)ELi(\d+)E", k[".name"])
        if not m:
            continue
        weight_grad, tile = m[1] == "1", (int(m[2]), int(m[3]))
        groups = {(256, 256): 1, (128, 128): 2, (128, 64): 3 if weight_grad else 2}[tile]
        assert k[".group_segment_fixed_size"] * groups <= LDS and k[".vgpr_count"] * groups <= REGISTERS, k[".name"]
        assert k[".vgpr_spill_count"] == 0 and k[".private_segment_fixed_size"] == 0, k[".name"]
        seen += 1
    assert seen == 24
    few = [k for k in _kernels() if "few_rows_kernel" in k[".name"]]
    assert len(few) == 4 and all(k[".group_segment_fixed_size"] * 2 <= LDS and k[".vgpr_count"] * 2 <= REGISTERS for k in few)


def test_row_kernels_spill_in_the_widest_layer_norms_alone():
    """Four pieces a lane of 16-bit rows, backward with a mean's gradient."""
    for k in _kernels():
        if re.search(r"norm_(fwd|bwd)_|activation_bwd_kernel|column_sum_kernel|pad_rows_kernel|gemm_join_kernel", k[".name"]):
            widest = re.search(r"norm_bwd_kernelILi[01]ELi\dELi\dELi0ELi0ELi4E", k[".name"])
            assert widest or k[".vgpr_spill_count"] == 0, k[".name"]
