"""The build's switch against packed float32 instructions: that it works on the device pass, and that nothing else is kept quiet."""
import pytest

from detectron_pytorch_amd import build


def without_the_feature(name=None):
    f = build.flags()
    at = f.index("-packed-fp32-ops")
    return f[:at] + [name] + f[at + 1:] if name else f[:at - 3] + f[at + 1:]


def test_the_switch_reaches_the_device_pass():
    build.check_no_packed_fp32(build.flags())


@pytest.mark.parametrize("name", [None, "-packed-fp32-op"])
def test_a_switch_that_does_nothing_is_an_error(name):
    with pytest.raises(RuntimeError, match="packed"):
        build.check_no_packed_fp32(without_the_feature(name))


def test_only_the_one_known_line_is_kept_quiet():
    known = "'-packed-fp32-ops' is not a recognized feature for this target (ignoring feature)"
    other = ["'-packed-fp32-op' is not a recognized feature for this target (ignoring feature)",
             "'+packed-fp32-ops' is not a recognized feature for this target (ignoring feature)", "warning: unused variable 'packed-fp32-ops'"]
    assert build.worth_saying("\n".join([known, other[0], known, *other[1:], known])) == other
    assert build.worth_saying(known + "\n\n") == []
