"""Layer norm over enough rows that the rings of bulk copies wrap, in each of their variants."""
import pytest
import torch

import manifold_b200 as gfn
from tests.test_gpu_norm import _run

# rows off 16 bytes and enough of them that the ring of bulk copies wraps, for each number of warps per row:
# forward and backward, the first sizes of each variant and the last
RING = [(8195, 99), (4099, 130), (9001, 511), (20011, 1001), (9001, 2047), (4099, 4095)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", RING, ids=str)
def test_layer_norm_of_many_rows_off_16_bytes(shape, dtype):
    _run(shape, dtype, torch.float32, seed=shape[1])
    assert gfn.cuda.ops.device_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(8195, 128), (4099, 520), (20011, 1000), (9001, 2048), (2500, 4096), (1500, 8192)], ids=str)
def test_layer_norm_of_many_rows_on_16_bytes(shape):
    for dtype in (torch.float32, torch.bfloat16):
        _run(shape, dtype, dtype, seed=shape[1])
    assert gfn.cuda.ops.device_error() == 0
