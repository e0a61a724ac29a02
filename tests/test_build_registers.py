"""CPU: the build fails when a kernel that divides its registers among warps is
not compiled to the number that it divides."""

import sys

import pytest

from conftest import PKG

LOG = """ptxas info    : Compiling entry function '_ZN3q6w20quantize_rows_kernelEPKfllPhPfPd' for 'sm_100a'
ptxas info    : Used 40 registers, used 0 barriers
ptxas info    : Compiling entry function '_ZN3q6w5paged11rows_kernelILi64EfEEv' for 'sm_100a'
    40 bytes stack frame, 40 bytes spill stores, 40 bytes spill loads
ptxas info    : Used {} registers, used 1 barriers, 40 bytes cumulative stack size
ptxas info    : Compiling entry function '_ZN3q6w5paged17rows_merge_kernelILi64ELi256EEEv' for 'sm_100a'
ptxas info    : Used 40 registers, used 0 barriers
"""


def test_other_register_counts_stop_the_build(monkeypatch):
    monkeypatch.syspath_prepend(str(PKG))
    monkeypatch.delitem(sys.modules, "build", raising=False)
    import build

    build.check_split_registers(LOG.format(128))
    for other in (120, 136):
        with pytest.raises(RuntimeError, match="rows_kernel"):
            build.check_split_registers(LOG.format(other))
