"""The int8 quantiser and product where their values are delicate: clusters
that wait for room, tokens that hold no number, activations far below zero."""
import numpy as np
import pytest

import spmm24
from int8_problems import bits_to_f64
from test_gpu_int8 import _dev, _quantized, _random_bits

pytestmark = pytest.mark.gpu


def test_strips_beside_other_work(cuda_device):
    """Many clusters of eight CTAs, waiting for room beside another stream's
    kernels, again and again: the same rows every time."""
    import torch

    rows, cols = 509, 4104
    bits = _random_bits(rows, cols, False, 77)
    pad = np.zeros(((rows + 7) // 8 * 8, cols), dtype=np.uint16)
    pad[:rows] = bits
    x = _dev(pad.reshape(-1, 8, cols).transpose(0, 2, 1).reshape(-1), cuda_device)
    want_q, want_s = (torch.from_numpy(v).to(cuda_device) for v in _quantized(bits_to_f64(bits, False).reshape(rows, cols)))
    big = torch.randn(2048, 2048, device=cuda_device, dtype=torch.float16)
    other = torch.cuda.Stream(cuda_device)
    torch.cuda.synchronize(cuda_device)
    outs = []
    for _ in range(100):
        with torch.cuda.stream(other):
            big @ big
        outs.append(spmm24.quantize_int8(x, rows, cols, packed=True))
    torch.cuda.synchronize(cuda_device)
    for q, s in outs:
        assert torch.equal(q, want_q) and torch.equal(s, want_s)
