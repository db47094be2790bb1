"""Source rules of the serving kernels."""
import os
import re

import pytest

from iris_b200 import _native

KERNELS = {"rotary.cu": {"qk_norm_rope_kernel"}, "paged_cache.cu": {"pages_kernel"},
           "paged_attention.cu": {"paged_attention_kernel", "paged_join_kernel", "paged_join_long_kernel"}}


@pytest.mark.parametrize("name", sorted(KERNELS))
def test_kernels_that_start_early_read_after_the_wait_and_coherently(name):
    """Placed while the kernel in front drains, like the element-wise kernels: nothing they read may be taken for constant, and no
    parameter's memory is read before the wait."""
    path = os.path.join(os.path.dirname(_native.__file__), "csrc", "kernels", name)
    source = re.sub(r"//[^\n]*", "", open(path).read())
    assert not re.search(r"__restrict__|__ldg|__ldlu|ld\.global\.nc", source)
    kernels = re.findall(r"__global__[^;{]*?(\w+_kernel)\([^{]*?\)\s*\{(.*?)\n\}\n", source, re.S)
    assert {k[0] for k in kernels} == KERNELS[name]
    for kernel, body in kernels:
        before = body[:body.index("grid_dependency_wait();")]
        assert not re.search(r"p\.\w+\[|\*p\.|\*\s*reinterpret_cast<const[^>]*>\(p\.", before), kernel
        assert body.index("grid_dependency_wait();") < body.index("grid_dependency_launch();")
