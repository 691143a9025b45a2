"""The int8 extension on the CPU: the host prune and packer, the argument
checks of its entry points (no GPU work is reached), and its plans."""
import numpy as np
import pytest

import spmm24
from int8_problems import prune_int8


def _decode(vals, meta, M, K):
    """Values + metadata -> the dense matrix, read off the documented layout."""
    out = np.zeros((M, K), dtype=np.int8)
    v = vals.view(np.int8).reshape(M // 16, K // 32, 16, 16)
    m = meta.reshape(M // 16, K // 128, 16, 16)
    for r in range(M):
        for g in range(K // 4):
            k = 4 * g
            nib = int(m[r // 16, k // 128, r % 16, (g % 32) // 2]) >> (4 * (g & 1)) & 15
            i0, i1 = nib & 3, nib >> 2
            assert i0 < i1
            kept = v[r // 16, k // 32, r % 16, (k % 32) // 2:][:2]
            out[r, k + i0], out[r, k + i1] = kept
    return out


def _matrix(M, K, seed):
    a = np.random.default_rng(seed).integers(-128, 128, (M, K)).astype(np.int8)
    a[0, :8] = [-128, 127, -127, 1, 5, -5, 5, -5]  # 128 is the largest magnitude; ties keep the lower index
    a[1, :12] = [0, 0, 0, 0, 0, 7, 0, 0, -128, 0, 0, -128]
    return a


def test_prune_keeps_the_two_largest_magnitudes():
    M, K = 48, 256
    a = _matrix(M, K, 1)
    got = spmm24.prune_2of4_int8(a, M, K).reshape(M, K)
    assert np.array_equal(got, prune_int8(a, M, K))
    assert list(got[0, :8]) == [-128, 127, 0, 0, 5, -5, 0, 0]


@pytest.mark.parametrize("M,K", [(16, 128), (48, 384)])
def test_compress_round_trip(M, K):
    a = prune_int8(_matrix(M, K, 2), M, K)
    vals, meta = spmm24.compress_a_int8(a, M, K)
    assert np.array_equal(_decode(vals, meta, M, K), a)


def test_compress_keeps_minus_128():
    """0x80 is a zero of fp8 (-0) and a value of int8."""
    a = np.zeros((16, 128), dtype=np.int8)
    a[:, 0::4] = -128
    a[:, 3::4] = 1
    vals, meta = spmm24.compress_a_int8(a, 16, 128)
    assert np.array_equal(_decode(vals, meta, 16, 128), a)
    a[3, 5] = 9  # a third value in a group
    with pytest.raises(ValueError, match="not 2:4"):
        spmm24.compress_a_int8(a, 16, 128)


def test_packer_refusals():
    z = np.zeros(16 * 128, dtype=np.int8)
    with pytest.raises(ValueError):
        spmm24.compress_a_int8(z, 16, 64)
    with pytest.raises(ValueError):
        spmm24.compress_a_int8(z, 8, 128)
    with pytest.raises(ValueError):
        spmm24.prune_2of4_int8(z, 16, 6)
    with pytest.raises(TypeError):
        spmm24.compress_a_int8(z.view(np.uint8), 16, 128)
    L = spmm24._lib
    bad = spmm24.CUDA_ERROR_INVALID_VALUE
    assert L.spmm24_pack_a_int8_device(None, 0x1000, 16, 128, 2, 0x2000, 0x3000, None) == bad
    assert L.spmm24_pack_a_int8_device(None, 0x1000, 16, 64, 0, 0x2000, 0x3000, None) == bad
    assert L.spmm24_pack_a_int8_device(None, 0x1008, 16, 128, 0, 0x2000, 0x3000, None) == bad
    assert L.spmm24_pack_a_int8_device(None, 0, 16, 128, 0, 0x2000, 0x3000, None) == bad


def _launch(values=0x10000, b=0x20000, meta=0x30000, c=0x40000, M=256, N=16, K=256, **kw):
    return spmm24.launch_int8(None, values, b, meta, c, M, N, K, **kw)


@pytest.mark.parametrize("kw,why", [
    (dict(values=0), "null"), (dict(b=0), "null"), (dict(meta=0), "null"), (dict(c=0), "null"),
    (dict(M=0), "positive"), (dict(N=0), "positive"), (dict(K=0), "positive"),
    (dict(M=250), "multiple of 16"), (dict(K=192), "multiple of 128"), (dict(K=262144), "262144"),
    (dict(split_k=-1), "split_k"), (dict(values=0x10008), "aligned"), (dict(b=0x20004), "aligned"),
    (dict(meta=0x30001), "aligned"), (dict(c=0x40001), "aligned"),
    (dict(w_scale=0x50002), "scales"), (dict(x_scale=0x50001), "scales"),
    (dict(flags=8), "flag"), (dict(flags=16), "flag"), (dict(flags=1 << 12), "flag"),
    (dict(activation=9), "activation"), (dict(out_layout=5), "layout"), (dict(alpha=float("inf")), "alpha"),
    (dict(bias=0x50001), "bias"), (dict(c=0x40002, out_layout=1), "packed"),
])
def test_launch_refusals(kw, why):
    assert _launch(**kw) == spmm24.CUDA_ERROR_INVALID_VALUE
    assert why in spmm24._lib.spmm24_last_error().decode()


@pytest.mark.parametrize("kw,why", [
    (dict(x=0), "null"), (dict(q=0), "null"), (dict(scale=0), "null"), (dict(rows=0), "positive"),
    (dict(cols=-1), "positive"), (dict(flags=1), "flag"), (dict(layout=2), "layout"), (dict(x=0x1001), "aligned"),
    (dict(scale=0x3002), "aligned"), (dict(ld=99), "ld"), (dict(ld=-1), "ld"),
    (dict(layout=1, ld=100), "ld"), (dict(layout=1, cols=100), "multiple of 8"), (dict(layout=1, x=0x1008), "16-byte"),
    (dict(layout=1, q=0x2004), "8-byte"), (dict(cols=(1 << 30) + 8), "2^30"), (dict(cols=2**31 - 1), "2^30"),
    (dict(layout=1, cols=2**31 - 8), "2^30"),
])
def test_quantize_refusals(kw, why):
    a = dict(x=0x1000, rows=4, cols=104, ld=0, layout=0, flags=0, q=0x2000, scale=0x3000) | kw
    rc = spmm24._lib.spmm24_quantize_int8(None, a["x"], a["rows"], a["cols"], a["ld"], a["layout"], a["flags"], a["q"],
                                          a["scale"])
    assert rc == spmm24.CUDA_ERROR_INVALID_VALUE
    assert why in spmm24._lib.spmm24_last_error().decode()


def test_plans():
    decode = spmm24.select_config_int8(4096, 8, 4096)
    assert decode["stage_k"] == 256 and decode["tile_n"] == 16 and not decode["cta_pair"]
    # shallow ring: two CTAs on one SM, as the fp8 form has
    assert 2 * (decode["smem_bytes"] + 1024) <= 233472
    assert 2 * (spmm24.select_config_int8(4096, 32, 4096)["smem_bytes"] + 1024) <= 233472
    prefill = spmm24.select_config_int8(11008, 4096, 4096)
    assert prefill["cta_pair"] == 1 and (prefill["tile_m"], prefill["tile_n"]) in ((256, 256), (512, 224))
    with pytest.raises(ValueError):
        spmm24.select_config_int8(256, 16, 64)
