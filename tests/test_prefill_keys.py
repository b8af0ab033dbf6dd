"""Which keys a tile of queries reads, by the kernel's own arithmetic on the host."""

import os
import subprocess

import pytest

from pagedserve_amd.ops import library

HERE = os.path.dirname(os.path.abspath(__file__))


def test_no_key_is_read_that_no_query_sees(tmp_path):
    """Portions in front of, across and behind the end of the block table, under windows and chunks, in ranges: every key read
    is seen by a query of its tile and has an entry of the table that the block keeps."""
    try:
        hipcc = library._hipcc()
    except library.KernelLibraryError as error:
        pytest.skip(str(error))
    program = os.path.join(str(tmp_path), "check")
    subprocess.run([hipcc, "-x", "hip", f"--offload-arch={library.ARCH}", "--offload-host-only", "-O2", "-std=c++17",
                    "-I", library.SOURCE_DIR, os.path.join(HERE, "prefill_keys_check.cpp"), "-o", program], check=True)
    result = subprocess.run([program], stdout=subprocess.PIPE, text=True, timeout=100)
    assert result.returncode == 0, result.stdout
