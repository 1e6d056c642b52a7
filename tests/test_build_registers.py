"""The build refuses a compiler that gives the kernels whose warps hand registers on another number than they count on: at the build, not at each call."""
import pytest
from tenzo_b200 import build

ENTRY = """ptxas info    : Compiling entry function '_ZN2tz21{0}EEvNS_10TreeLaunchE14CUtensorMap_stS2_' for 'sm_100a'
ptxas info    : Function properties for _ZN2tz21{0}EEvNS_10TreeLaunchE14CUtensorMap_stS2_
    64 bytes stack frame, 196 bytes spill stores, 196 bytes spill loads
ptxas info    : Used {1} registers, used 16 barriers, 64 bytes cumulative stack size, 6400 bytes smem
"""


def log(**other):
    return "".join(ENTRY.format(k, other.get(k[-4:], v[0])) for k, v in build.LAUNCHED_REGISTERS.items())


def test_numbers_that_are_as_they_have_to_be():
    build.check_registers(log())
    build.check_registers(log(i64E=93))                                         # given out by eights: 96


@pytest.mark.parametrize("which,used", [("i64E", 88), ("i64E", 120), ("i48E", 120), ("i32E", 72), ("i16E", 255)])
def test_other_numbers_are_refused(which, used):
    with pytest.raises(RuntimeError, match="registers"):
        build.check_registers(log(**{which: used}))


def test_a_kernel_that_is_not_there_is_refused():
    with pytest.raises(RuntimeError):
        build.check_registers("")


def test_this_build():
    build.build()
    build.check_registers((build.PKG / "lib" / "ptxas.log").read_text())
