"""The code objects of the attention over 16 bits (CPU test: reads the library
file only): kernels for pages that are no multiple of 8, which form every
key's address in vector registers, hold a workgroup's share of the work in
scalar ones.  In vector registers it took 15 to 20 more, and 4 to 25% of the
time."""
import re

from test_codeobj import code_object_notes

MOST = {2: 128, 3: 168, 4: 184}  # by head_dim / 32: four and three waves a SIMD where that many fit, else what the loop takes


def registers(tmp_path):
    found = {}
    for text in code_object_notes(tmp_path):
        for block in re.split(r"\n  - \.", text):
            name = re.search(r"\.name:\s*\S*attend_kernelILi(\d)ELb([01])ELb0ELb([01])E", block)
            count = re.search(r"\.vgpr_count:\s*(\d+)", block)
            if name and count and int(name.group(1)) in MOST:
                found[name.groups()] = int(count.group(1))
    return found


def test_shares_take_no_vector_registers_where_addresses_do(tmp_path):
    found = registers(tmp_path)
    assert len(found) == 6, found  # three widths, two types (with such pages every width takes the form for any head_dim)
    assert all(n <= MOST[int(k[0])] for k, n in found.items()), found
