"""The mixture-of-experts layer at sizes whose workgroups take more columns and more tokens at a time, with ragged ends in every direction; many experts with few tokens
each; K split between workgroups with few."""
import pytest

from test_gpu_moe import Layer

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hidden,inter,experts,top,tokens", ((1376, 672, 24, 6, (64, 33)),   # 128 columns, 32 tokens at a time
                                                            (1376, 672, 24, 6, (17, 6)),     # 128 columns, 16 tokens
                                                            (224, 1056, 2, 1, (64, 50)),     # 64 columns, 32 tokens, K split
                                                            (160, 2304, 4, 2, (16, 1)),
                                                            (64, 96, 600, 8, (64, 9)),
                                                            (96, 64, 1024, 64, (3, 64))))
def test_layers(gpu, hidden, inter, experts, top, tokens):
    layer = Layer(hidden + experts, hidden, inter, experts)
    for t in tokens:
        layer.check(gpu, "device", t, top, beta=1.0)
