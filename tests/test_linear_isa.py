"""The tiled product of frhip_linear keeps the rule of the product kernels that it shares its loading waves with: no LDS read of its
multiplying waves is outstanding at a bare barrier, behind which that LDS is written again."""
import re
import subprocess

import pytest

from test_kernel_isa import LIB, OBJDUMP, code_objects, functions, reads_outstanding_at_barriers


@pytest.mark.skipif(OBJDUMP is None, reason="no llvm-objdump")
def test_no_fragment_read_of_the_linear_tiles_is_outstanding_at_a_barrier(tmp_path):
    seen = 0
    for i, obj in enumerate(code_objects(open(LIB, "rb").read())):
        if b"linear_ring_kernel" not in obj:  # one object holds all of them
            continue
        path = tmp_path / ("%d.co" % i)
        path.write_bytes(obj)
        listing = subprocess.run([OBJDUMP, "-d", "--mcpu=gfx950", str(path)], capture_output=True, text=True, check=True).stdout
        for name, body in functions(listing).items():
            if re.search("linear_(ring|wide|q8)_kernel", name):
                assert any(t == "s_barrier" for _, t, _ in body) and any("mfma" in t for _, t, _ in body), name
                assert not reads_outstanding_at_barriers(body), name
                seen += 1
    assert seen == 10  # tiles of 64, 128 (two depths) and 256 rows, K with and without a rest; uint8: 64 and 128 rows
