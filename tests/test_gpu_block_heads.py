"""MI355X: attention over so many small graphs that a workgroup goes over several key heads, one after the other, at the head sizes
whose kernels put registers away: what belongs to a thread has to be there for the second head too."""
import pytest
import torch

from tests.test_gpu_block_ops import TYPES, attention_case, attention_run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("dim", [72, 128])
@pytest.mark.parametrize("dtype", TYPES)
def test_attention_over_several_key_heads_a_workgroup(dtype, dim, masked):
    c = attention_case([(7 * i) % 4 for i in range(2200)], None, 4, 2, dim, dtype, masked, extra=1)
    attention_run(*c, same=True)
