"""Products with integer 4-bit weights for more rows than one pass over the codes takes: a prompt's, in one matrix and in uneven groups, through an index and as they lie, on the stream
over the codes and on the kernel for any layout."""
import numpy as np
import pytest

from test_gpu_gemm_grouped import split
from test_gpu_gemm_u4 import run_u4

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shift", (0, 1), ids=("stream", "any layout"))
@pytest.mark.parametrize("kind", ("bf16", "f16"))
def test_a_prompt(gpu, kind, shift):
    run_u4(gpu, kind, kind, 1100, 136, 512, 128, fronts=(0, shift), seed=1)
    run_u4(gpu, kind, "f32", 1031, 40, 288, 32, zeros=None, alpha=0.5, beta=-1.0, fronts=(0, shift), seed=2)


@pytest.mark.parametrize("shift", (0, 1), ids=("stream", "any layout"))
@pytest.mark.parametrize("kind", ("bf16", "f16"))
def test_a_prompt_in_uneven_groups(gpu, kind, shift):
    rng = np.random.default_rng(3)
    offsets = np.concatenate(([0], np.cumsum([1, 0, 700, 33, 32, 31, 0, 517, 2]))).astype(np.int32)
    index = rng.integers(0, 400, 1330)
    index[rng.random(1330) < 0.05] = -1
    run_u4(gpu, kind, kind, 1330, 72, 256, 64, offsets, 9, index=index, a_rows=400, fronts=(0, shift), seed=4)
    run_u4(gpu, kind, "f32", 2005, 40, 384, 128, split(rng, 2000, 20), 20, zeros="far", fronts=(0, shift), seed=5)
