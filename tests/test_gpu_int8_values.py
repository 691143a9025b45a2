"""The int8 quantiser and product where their values are delicate: clusters
that wait for room, tokens that hold no number, activations far below zero."""
import numpy as np
import pytest

import spmm24
from act_values import act_tails
from int8_problems import bits_to_f64, problem
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


# every kernel of the product, and a shape that it takes
KERNELS = {"cluster": (dict(pair=0), 528, 269, 256), "cluster16": (dict(pair=0, tile_n=16), 528, 40, 256),
           "pair": (dict(pair=1, pair2=0, pair_split=1), 528, 269, 256),
           "pair-split": (dict(pair=1, pair2=0, pair_split=2), 528, 269, 512),
           "pair2": (dict(pair=1, pair2=1), 1040, 269, 256), "persistent": (dict(pair2=1), 5120, 2048, 256)}


def _product(device, M, N, K, seed):
    """(values, metadata, B, exact sums) of a problem on the device."""
    import torch

    a, b = problem(M, N, K, seed)
    vals, meta = spmm24.compress_a_int8(a, M, K)
    acc = torch.from_numpy(a).to(device).double() @ torch.from_numpy(b).to(device).double().T
    return _dev(vals, device), _dev(meta, device), _dev(b, device), acc


@pytest.mark.parametrize("act", [0, 1, 2, 3], ids=["none", "relu", "silu", "gelu"])
@pytest.mark.parametrize("kernel", list(KERNELS))
@pytest.mark.parametrize("packed", [False, True], ids=["rows", "strips"])
def test_a_token_that_holds_no_number_stays_so(cuda_device, tuning, kernel, act, packed):
    """Infinite and NaN scales (the quantiser's for such rows): their columns are NaN, whatever the activation."""
    import torch

    kw, M, N, K = KERNELS[kernel]
    tuning(**kw)
    vals, meta, b, _ = _product(cuda_device, M, N, K, 3)
    bad = [0, 7, 21, N - 1]
    scale = torch.full((N,), 2.0 ** -13, device=cuda_device)
    scale[bad] = torch.tensor([float("nan"), float("inf"), float("nan"), float("inf")], device=cuda_device)
    b = b.clone()
    b[bad] = 0  # as the quantiser writes them: 0 * inf
    strips = (N + 7) // 8
    c = torch.zeros(strips * 8 * M, dtype=torch.float16, device=cuda_device)
    bias = torch.ones(M, dtype=torch.float16, device=cuda_device)
    rc = spmm24.launch_int8(torch.cuda.current_stream(cuda_device), vals, b, meta, c, M, N, K, x_scale=scale, bias=bias,
                            activation=act, out_layout=spmm24.OUT_PACKED_B if packed else spmm24.OUT_ROW_MAJOR)
    assert rc == 0
    y = c.reshape(strips, M, 8).transpose(0, 1).reshape(M, -1)[:, :N] if packed else c[: M * N].reshape(M, N)
    nan = torch.isnan(y)
    assert nan[:, bad].all() and int(nan.sum()) == M * len(bad)


@pytest.mark.parametrize("act", [2, 3], ids=["silu", "gelu"])
@pytest.mark.parametrize("bf16", [False, True], ids=["fp16", "bf16"])
@pytest.mark.parametrize("kernel", list(KERNELS))
def test_activations_below_zero(cuda_device, tuning, kernel, bf16, act):
    """Pre-activations within 100 of zero, most of them in -20 .. 20, exact in fp32 (powers of two for scales), against
    the value itself: far below zero the activation is small, and its error has to be small beside it.

    Bound, relative to the value: e^-x by the fast exponential 2 + 1.17 |x| steps of 2^-23, 1 + e half a one, the
    fast division 2, the product with y half a one: (5 + 1.2 |x|) 2^-23.  GELU's x is itself the end of seven roundings
    (two of them its constants) of 2^-24, which move e^-x by 3.5 |x| 2^-23.  Then half a step of C's type."""
    import torch

    kw, M, N, K = KERNELS[kernel]
    tuning(**kw)
    vals, meta, b, acc = _product(cuda_device, M, N, K, 5)
    step = 2.0 ** -13 if K == 256 else 2.0 ** -14
    c = torch.zeros(M, N, dtype=torch.bfloat16 if bf16 else torch.float16, device=cuda_device)
    rc = spmm24.launch_int8(torch.cuda.current_stream(cuda_device), vals, b, meta, c, M, N, K, flags=spmm24.BF16 if bf16 else 0,
                            x_scale=torch.full((N,), step, device=cuda_device), activation=act)
    assert rc == 0
    pre = acc * step
    assert (pre < -8).any() and (pre > 8).any() and pre.abs().max() < 100
    ref, x = act_tails(pre, act)
    half, tiny = (2.0 ** -8, 2.0 ** -134) if bf16 else (2.0 ** -11, 2.0 ** -25)
    # x is capped where the value is below every subnormal of C's type
    rel = (5 + (1.2 if act == 2 else 4.7) * x.clamp(max=110)) * 2.0 ** -23
    off = (c.double() - ref).abs()
    tol = ref.abs() * (half + rel * (1 + half)) + tiny
    assert (off <= tol).all(), float((off / tol).max())
