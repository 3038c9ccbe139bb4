"""CPU: the flags that a kernel's first call on a device sets are atomic.  Host threads may make
that call at the same time: the binding calls without the interpreter's lock."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "gpu-kernels_b200", "csrc")


@pytest.mark.parametrize("name", ["embedding", "logprobs", "moe", "moe_layer", "moe_products"])
def test_first_call_flags_are_atomic(name):
    with open(os.path.join(CSRC, name + ".cu")) as f:
        flags = re.findall(r"^ +static (?!constexpr|const |__device__)(.*?)[;=]", f.read(), re.M)
    assert flags and all(flag.startswith("std::atomic<") for flag in flags), flags
