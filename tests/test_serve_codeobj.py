"""The serving kernels' code objects (CPU test: reads the library file only).

Their dynamic LDS arrays are read and written as 16-byte vectors and start
where the kernel's fixed LDS ends: it has to be a multiple of 16 bytes."""
import re

from test_codeobj import code_object_notes


def test_dynamic_lds_of_the_serving_kernels_starts_at_a_vector(tmp_path):
    sizes = {}
    for text in code_object_notes(tmp_path):
        for block in re.split(r"\n  - \.", text):
            name = re.search(r"\.name:\s*(\S*(?:attend|adapter_down|adapter_up)_kernel\S*)", block)
            fixed = re.search(r"\.group_segment_fixed_size:\s*(\d+)", block)
            if name and fixed:
                sizes[name.group(1)] = int(fixed.group(1))
    for family in ("attend_kernel", "adapter_down_kernel", "adapter_up_kernel"):
        assert any(family in n for n in sizes), f"no {family} in the code objects"
    odd = {n: s for n, s in sizes.items() if s % 16}
    assert not odd, f"{len(odd)} kernels, among them {list(odd.items())[:2]}"
