"""The code objects of the kernels over a cache in 4 bits (CPU test: reads the
library file only): the attention's dynamic LDS is read and written as 16-byte
vectors and starts where its fixed LDS ends, a multiple of 16 bytes."""
import re

from test_codeobj import code_object_notes


def test_dynamic_lds_of_the_int4_attention_starts_at_a_vector(tmp_path):
    sizes = {}
    for text in code_object_notes(tmp_path):
        for block in re.split(r"\n  - \.", text):
            name = re.search(r"\.name:\s*(\S*attend4_kernel\S*)", block)
            fixed = re.search(r"\.group_segment_fixed_size:\s*(\d+)", block)
            if name and fixed:
                sizes[name.group(1)] = int(fixed.group(1))
    assert sizes, "no attend4_kernel in the code objects"
    odd = {n: s for n, s in sizes.items() if s % 16}
    assert not odd, f"{len(odd)} kernels, among them {list(odd.items())[:2]}"
